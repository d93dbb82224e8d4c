"""What the Python calls of the 8-bit cache and of sampling hand to the library, without a GPU:
the tensors are on the CPU, the library is a record of its calls."""
import types

import pytest

import gcu

torch = pytest.importorskip("torch")


class Calls:
    """A library that launches nothing: every call is noted and succeeds."""

    def __init__(self, work=0):
        self.made, self.work = [], work

    def __getattr__(self, name):
        def call(*args, **kw):
            if name.endswith("_work"):
                return self.work
            self.made.append((name, args))
            return 0
        return call


@pytest.fixture
def library(monkeypatch):
    calls = Calls()
    gcu._torch()
    monkeypatch.setattr(gcu, "lib", lambda: calls)
    monkeypatch.setattr(gcu, "_device", lambda what, index: -1)
    monkeypatch.setattr(gcu, "_on", lambda stream, dev: 0)
    return calls


def sample(logits):
    m = logits.shape[0]
    gcu.dev_sample(torch.zeros(m, dtype=torch.int32), logits, torch.zeros(m))


def test_logits_rows_that_are_one_row(library):
    """A stride of 0 is not the library's 0, which stands for rows one behind the other."""
    one = torch.zeros((1, 40))
    sample(one)
    sample(one.expand(3, -1).contiguous())
    assert len(library.made) == 2
    for rows in (one.expand(3, -1), torch.zeros(60).as_strided((3, 40), (8, 1))):
        with pytest.raises(gcu.GcuError, match="rows of 40 logits"):
            sample(rows)
    assert len(library.made) == 2


def prefill(xo, ntok, nh=2, hd=64):
    kv = gcu.KvCacheI8.empty(1, 1, 16, hd, device="cpu")
    gcu.dev_attention_prefill_i8(xo, torch.zeros((nh, ntok, hd)), kv, 0)


def test_prefill_rows_that_are_one_row(library):
    """As above for the rows that prefill attention writes."""
    prefill(torch.zeros((3, 128)), 3)
    prefill(torch.zeros((3, 160))[:, :128], 3)
    prefill(torch.zeros((1, 128)).expand(1, -1), 1)
    assert [args[1] for _, args in library.made] == [128, 160, 0]
    for xo in (torch.zeros((1, 128)).expand(3, -1), torch.zeros(300).as_strided((3, 128), (64, 1))):
        with pytest.raises(gcu.GcuError, match="rows"):
            prefill(xo, 3)
    assert len(library.made) == 3


BIG = (1 << 32) + 3  # 3 in a C int


def test_numbers_past_32_bits(library):
    """The library's counts are C ints; a larger one does not wrap to another count."""
    kv = gcu.KvCacheI8.empty(1, 1, 16, 64, device="cpu")
    f32 = lambda *shape: torch.zeros(shape)
    x, xq, rows = f32(1, 2, 64), f32(2, 3, 64), f32(3, 128)
    calls = [
        lambda n: gcu.dev_sample(torch.zeros(1, dtype=torch.int32), f32(1, 8), f32(1), top_k=n),
        lambda n: gcu.dev_attention_decode_i8(f32(1, 2, 64), x, kv, None, n, 1.0),
        lambda n: gcu.dev_attention_decode_i8(f32(1, 2, 64), x, kv, None, 8, 1.0, slide=n),
        lambda n: gcu.dev_attention_decode_i8(f32(1, 2, 64), x, kv, None, 8, 1.0, prefix=kv, plen=n),
        lambda n: gcu.dev_attention_prefill_i8(rows, xq, kv, n),
        lambda n: gcu.dev_attention_prefill_i8(rows, xq, kv, 0, slide=n),
        lambda n: gcu.dev_cache_i8_read(f32(1, 1, 2, 64), f32(1, 1, 2, 64), kv, n),
        lambda n: gcu.dev_qkv_norm_rope_cache_i8(xq, f32(3, 256), kv, f32(3, 64), n),
    ]
    for call in calls:
        call(3)
        call(-1)  # in range here; the library says what it thinks of it
        made = len(library.made)
        for n in (BIG, 1 << 31, -BIG):
            with pytest.raises(gcu.GcuError, match="32 bits"):
                call(n)
        assert len(library.made) == made


class Streams:
    """Stands for torch.cuda.stream: which stream is the current one."""

    def __init__(self, monkeypatch):
        self.current, self.allocated = None, []
        for name in ("empty", "zeros", "ones"):
            monkeypatch.setattr(torch, name, self.noting(getattr(torch, name)))
        monkeypatch.setattr(torch.cuda, "stream", self.use)

    def noting(self, make):
        def noted(*args, **kw):
            self.allocated.append(self.current)
            return make(*args, **kw)
        return noted

    def use(self, stream):
        outer = self

        class Context:
            def __enter__(self):
                self.before, outer.current = outer.current, stream

            def __exit__(self, *exc):
                outer.current = self.before
        return Context()


def test_scratch_belongs_to_the_stream_that_uses_it(library, monkeypatch):
    """Taken from another stream's pool, a block could still be in use there."""
    library.work = 1 << 12
    kv = gcu.KvCacheI8.empty(1, 1, 16, 64, device="cpu")
    x, xo, rows, xq = torch.zeros((1, 2, 64)), torch.zeros((1, 2, 64)), torch.zeros((3, 128)), torch.zeros((2, 3, 64))
    side = types.SimpleNamespace(cuda_stream=7)
    streams = Streams(monkeypatch)
    monkeypatch.setattr(gcu, "_on", lambda stream, dev: (stream or streams.current or types.SimpleNamespace(cuda_stream=0)).cuda_stream)
    for stream in (None, side):
        gcu.dev_attention_decode_i8(xo, x, kv, None, 8, 1.0, stream=stream)
        gcu.dev_attention_prefill_i8(rows, xq, kv, 0, stream=stream)
    assert streams.allocated == [None, None, side, side] and streams.current is None


def test_sampled_tokens_belong_to_the_stream_that_writes_them(library, monkeypatch):
    """And are not handed out again while the stream that was current may still read them."""
    import decode
    dec = object.__new__(decode.Decoder)
    dec.torch, dec.dev, dec.logits, dec.slogits = torch, "cpu", torch.zeros((1, 8)), torch.zeros((3, 8))
    side, readers = object(), []
    u = torch.zeros(1), torch.zeros(3)
    streams = Streams(monkeypatch)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: readers.append(s))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: streams.current)
    assert dec.sample(u[0]).shape == (1,)
    assert dec.sample(u[1], seqs=True, stream=side).shape == (3,)
    assert streams.allocated == [None, side] and readers == [None] and streams.current is None


def test_a_fork_is_made_on_the_stream_that_steps_it(monkeypatch):
    """Its caches are filled, and the last fork's dropped, in the order of that stream."""
    import decode
    dec = object.__new__(decode.Decoder)
    dec.torch, dec.dev, dec.kv_bits, dec.clen = torch, "cpu", 8, 16
    dec.cfg = dict(nl=2, n_heads=2, nkv=1, hdim=64, dim=32, mlp_dim=48, nvocab=10)
    dec.L = [{w: (torch.zeros((4, 32), dtype=torch.int8), torch.zeros(4)) for w in ("wq", "wk", "wv")}] * 2
    streams, side = Streams(monkeypatch), object()
    dec.fork(3, 4, 5)
    assert set(streams.allocated) == {None}
    del streams.allocated[:]
    dec.fork(3, 4, 5, stream=side)
    assert set(streams.allocated) == {side} and streams.current is None
    streams.copies = []
    copy = torch.Tensor.copy_
    monkeypatch.setattr(torch.Tensor, "copy_", lambda *a, **k: streams.copies.append(streams.current) or copy(*a, **k))
    for s in (None, side):
        dec.set_seq_freqs(torch.zeros((3, 64)).numpy(), torch.ones((3, 64)).numpy(), stream=s)
    assert streams.copies == [None, side]


def test_steps_past_the_tail_are_refused(monkeypatch):
    """Not carried out with the sequence's attention left out."""
    import decode
    dec = object.__new__(decode.Decoder)
    dec.torch, dec.dev, dec.kv_bits, dec.clen = torch, "cpu", 8, 16
    dec.cfg = dict(nl=1, n_heads=2, nkv=1, hdim=64, dim=32, mlp_dim=48, nvocab=10, q_scale=64.0, eps=1e-6, swa=[0],
                   qk_norm=0, mlp_pre=0, mlp_pst=0, slide=0, sc_att=0.0, sc_log=0.0)
    w = (torch.zeros((4, 32), dtype=torch.int8), torch.zeros(4))
    dec.L = [dict({k: w for k in ("wq", "wk", "wv", "wo", "w1", "w2", "w3")}, n1=None, n2=None)]
    dec.emb, dec.fnorm, dec.kv8 = w, None, [gcu.KvCacheI8.empty(1, 1, 16, 64, "cpu")]
    dec.fork(3, 4, 2)
    calls = Calls()
    monkeypatch.setattr(decode, "gcu", calls)
    for _ in range(2):
        dec.step_seqs()
    made = len(calls.made)
    for _ in range(2):
        with pytest.raises(ValueError, match="2 tokens"):
            dec.step_seqs()
    assert len(calls.made) == made and dec.slen.tolist() == [2, 2, 2]
    dec.slen.copy_(torch.tensor([-1, 1, 0]))  # one is done, the others go back
    dec.step_seqs()
    assert dec.slen.tolist() == [-1, 2, 1]
    with pytest.raises(ValueError, match="2 tokens"):
        dec.step_seqs()
    dec.slen[1] = -1
    dec.step_seqs()
    assert dec.slen.tolist() == [-1, -1, 2]
    monkeypatch.setattr(decode, "gcu", gcu)
    dec.fork(1, 4, 1)
    monkeypatch.setattr(decode, "gcu", calls)
    dec.step_seqs()
    assert dec.slen.tolist() == [1]


def test_writes_to_one_buffer_for_keys_and_values():
    """A cache that is only read may have them in one; written, each would overwrite the other."""
    import ctypes
    from test_i8_host import P, kv_struct, refused
    kv = kv_struct()
    assert kv.k == kv.v
    lib, ref = gcu.lib(), ctypes.byref
    other = torch.zeros(4096, dtype=torch.int8)
    at = (other.data_ptr() + 15) // 16 * 16
    for over in ({}, dict(v=at), dict(vs=at)):
        c = kv_struct(**over)
        q = torch.zeros(2048)
        qkv = (q.data_ptr() + 15) // 16 * 16
        refused(lib.gcu_dev_qkv_norm_rope_cache_i8(P, qkv, 512, ref(c), None, None, 1e-6, P, 1.0, 4, 0, 1, None), "k and v")
        refused(lib.gcu_dev_qkv_norm_rope_cache_i8_seqs(P, qkv, 512, ref(c), P, None, None, 1e-6, P, 1.0, 4, None), "k and v")
