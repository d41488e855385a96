"""Key / value cache entry points without a GPU: sizes, refusals (every call below fails before a pointer is
used or a kernel launched), and the definition's restatement against itself."""
import ctypes

import numpy as np
import pytest

import kv_cache_ref as ref
from example_matmul_metal4_b200 import _lib

FAKE = 1 << 20  # a stand-in address, 16-byte aligned
INVALID, UNSUPPORTED = _lib.MM4_ERR_INVALID, _lib.MM4_ERR_UNSUPPORTED


def _plan(**kw):
    d = dict(pages=7, page_size=64, heads_q=8, heads_kv=2, head_dim=128, bits=4, causal=1, scale=0.0)
    d.update(kw)
    h = ctypes.c_void_p()
    rc = _lib.lib().mm4_kv_cache_plan_create(ctypes.byref(h), ctypes.byref(_lib.KVCacheDesc(*d.values())))
    return rc, h


def _batch(**kw):
    d = dict(sequences=3, tokens=5, max_new=2, pages_per_sequence=4, page_table=FAKE, lengths=FAKE, offsets=FAKE)
    d.update(kw)
    return _lib.KVCacheBatchDesc(*d.values())


@pytest.mark.parametrize("D,bits,row", [(128, 4, 80), (128, 8, 144), (64, 4, 40), (64, 8, 72)])
def test_sizes(D, bits, row):
    L = _lib.lib()
    rc, h = _plan(head_dim=D, bits=bits, page_size=32, heads_kv=4, pages=1 << 20)
    assert rc == 0 and ref.row_bytes(D, bits) == row
    assert L.mm4_kv_cache_page_bytes(h) == 4 * 2 * 32 * row
    assert L.mm4_kv_cache_bytes(h) == (4 * 2 * 32 * row) << 20
    L.mm4_kv_cache_plan_destroy(h)
    assert L.mm4_kv_cache_page_bytes(None) == 0 and L.mm4_kv_cache_bytes(None) == 0
    assert L.mm4_kv_cache_attention_workspace_size(None, None) == 0
    L.mm4_kv_cache_plan_destroy(None)


@pytest.mark.parametrize("kw,rc", [
    (dict(pages=0), INVALID), (dict(pages=1 << 31), UNSUPPORTED), (dict(page_size=48), INVALID),
    (dict(page_size=8), INVALID), (dict(page_size=512), INVALID), (dict(heads_q=0), INVALID),
    (dict(heads_kv=3), INVALID), (dict(heads_kv=-1), INVALID), (dict(head_dim=96), UNSUPPORTED),
    (dict(head_dim=0), INVALID), (dict(bits=3), INVALID), (dict(causal=2), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(heads_q=8192, heads_kv=8192), UNSUPPORTED)])
def test_plan_refusals(kw, rc):
    got, h = _plan(**kw)
    assert got == rc and not h
    assert _lib.lib().mm4_last_error()


def test_null_plan_arguments():
    L = _lib.lib()
    assert L.mm4_kv_cache_plan_create(None, None) == INVALID
    h = ctypes.c_void_p()
    assert L.mm4_kv_cache_plan_create(ctypes.byref(h), None) == INVALID


def _calls(L, h):
    """name -> call(batch reference, pointers, strides): K / V of width 256, Q / O of width 1024."""
    return {
        "append": lambda b, p, s: L.mm4_kv_cache_append(h, b, p[0], s[0], p[1], s[1], p[2], None),
        "read": lambda b, p, s: L.mm4_kv_cache_read(h, b, p[2], p[0], s[0], p[1], s[1], None),
        "attention": lambda b, p, s: L.mm4_kv_cache_attention(h, b, p[0], s[0], p[2], p[1], s[1], None, FAKE, 1 << 40,
                                                              None),
    }


@pytest.mark.parametrize("name,width", [("append", 256), ("read", 256), ("attention", 1024)])
def test_call_refusals(name, width):
    L = _lib.lib()
    rc, h = _plan()
    assert rc == 0
    call = _calls(L, h)[name]
    good = ([FAKE] * 3, [width, width])
    assert _calls(L, None)[name](ctypes.byref(_batch()), *good) == INVALID
    assert call(None, *good) == INVALID
    for kw in (dict(sequences=-1), dict(tokens=-1), dict(max_new=-1), dict(pages_per_sequence=-1),
               dict(page_table=None), dict(lengths=None), dict(offsets=None), dict(lengths=FAKE + 2)):
        assert call(ctypes.byref(_batch(**kw)), *good) == INVALID, kw
    assert call(ctypes.byref(_batch(pages_per_sequence=1 << 25)), *good) == UNSUPPORTED
    for i in range(3):
        for bad in (None, FAKE + 8):
            p = [FAKE] * 3
            p[i] = bad
            assert call(ctypes.byref(_batch()), p, good[1]) == INVALID, (i, bad)
    for i in range(2):
        for bad in (width - 8, width + 4, 0, -width):
            s = [width, width]
            s[i] = bad
            assert call(ctypes.byref(_batch()), good[0], s) == INVALID, (i, bad)
    # nothing to do: no row, no sequence; no pointer is looked at
    assert call(ctypes.byref(_batch(tokens=0)), [None] * 3, [0, 0]) == 0
    assert call(ctypes.byref(_batch(sequences=0)), [None] * 3, [0, 0]) == 0
    if name == "attention":
        assert call(ctypes.byref(_batch(max_new=0)), *good) == INVALID
        assert b"max_new" in L.mm4_last_error()
        assert L.mm4_kv_cache_attention(h, ctypes.byref(_batch()), FAKE, width, FAKE, FAKE, width, FAKE + 2, FAKE,
                                        1 << 40, None) == INVALID
    L.mm4_kv_cache_plan_destroy(h)


def test_python_wrapper_refusals():
    import torch

    from example_matmul_metal4_b200.kv_cache import KVCacheBatch, KVCacheDimensions, KVCachePlan
    with pytest.raises(_lib.MM4Error):
        KVCachePlan(KVCacheDimensions(4, 64, 8, 3, 128))
    plan = KVCachePlan(KVCacheDimensions(4, 64, 8, 2, 128))
    assert plan.cacheBytes == 4 * plan.pageBytes
    assert plan.allocate("cpu").shape == (4, plan.pageBytes)
    i32 = torch.int32
    with pytest.raises(ValueError, match="CUDA int32"):
        KVCacheBatch(torch.zeros(1, 1, dtype=i32), torch.zeros(1, dtype=i32), torch.zeros(2, dtype=i32), 1, 1)


def test_restatement_rounds_scales_towards_zero_and_inverts():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 128)).astype(np.float16)
    for bits in (4, 8):
        codes, scale, zero = ref.quantise(x, bits)
        top = 2 ** bits - 1
        g = x.astype(np.float64).reshape(50, 4, 32)
        span = g.max(-1) - g.min(-1)
        assert (scale.astype(np.float64) * top <= span * (1 + 2.0 ** -23)).all()
        assert codes.max() <= top
        back = ref.unpack(ref.pack(x, bits), 128, bits)
        assert np.array_equal(back, ref.values(codes, scale, zero))
        err = np.abs(back.astype(np.float64) - x).reshape(50, 4, 32).max(-1)
        assert (err <= span / top / 2 + span * 2.0 ** -10 + 4 * 2.0 ** -11).all()


def test_attention_form_by_sizes():
    """The kernel is chosen from the batch's sizes: rows of a key / value head in one sequence (max_new times the
    group of 4 here), the tokens a sequence can hold and the number of units."""
    L = _lib.lib()
    rc, h = _plan()
    assert rc == 0

    def form(**kw):
        b = _batch(**kw)
        return (L.mm4_kv_cache_attention_kernel_name(h, ctypes.byref(b)),
                L.mm4_kv_cache_attention_workspace_size(h, ctypes.byref(b)))

    assert form(max_new=2) == (b"kv_attention_few<8 rows, team>", 0)
    assert form(max_new=3) == (b"kv_attention_few<16 rows, team>", 0)
    assert form(max_new=2, pages_per_sequence=32) == (b"kv_attention_few<8 rows, team>", 0)
    name, ws = form(max_new=2, pages_per_sequence=33)
    assert name == b"kv_attention_few<8 rows, split>" and ws > 0
    assert form(max_new=2, sequences=75)[0] == b"kv_attention_few<8 rows, split>"
    for new in (5, 12):
        name, ws = form(max_new=new)
        assert name == b"kv_attention_few<24 rows, split>" and ws > 0
    name, ws = form(max_new=13)
    assert name == b"kv_attention_many" and ws >= 2 * 148 * 256 * (128 + 2) * 4
    assert form(tokens=0)[1] == 0 and form(sequences=0)[1] == 0
    # a workspace that is missing, too small or misaligned
    b = _batch(max_new=13)
    args = (FAKE, 1024, FAKE, FAKE, 1024, None)
    assert L.mm4_kv_cache_attention(h, ctypes.byref(b), *args, None, ws, None) == _lib.MM4_ERR_WORKSPACE
    assert L.mm4_kv_cache_attention(h, ctypes.byref(b), *args, FAKE, ws - 1, None) == _lib.MM4_ERR_WORKSPACE
    assert L.mm4_kv_cache_attention(h, ctypes.byref(b), *args, FAKE + 8, ws, None) == INVALID
    b = _batch(max_new=1 << 28, tokens=1 << 30)
    assert L.mm4_kv_cache_attention(h, ctypes.byref(b), *args, FAKE, 1 << 40, None) == UNSUPPORTED
    L.mm4_kv_cache_plan_destroy(h)


def test_exact_division_by_the_code_range():
    """x / 15 and x / 255 in fp32 by a product, its remainder and a correction (Markstein) equal the division, for
    the differences of fp16 values that a group's range can be: all bit patterns of one sign against a few."""
    f = np.float32
    v = np.arange(0, 0x7C00, dtype=np.uint16).view(np.float16).astype(f)
    for other in (0.0, 2.0 ** -24, 0.333, 1.0, 1000.5, 65504.0):
        x = np.abs(v - f(np.float16(other))).astype(f)
        x = np.concatenate([x, (v + f(np.float16(other))).astype(f)])
        for top in (15, 255):
            inv = f(1) / f(top)
            q = (x * inv).astype(f)
            # float64 holds -q * top + x and q + r * inv to well below half a unit of the fp32 result
            r = (x.astype(np.float64) - q.astype(np.float64) * top).astype(f)
            got = (q.astype(np.float64) + r.astype(np.float64) * np.float64(inv)).astype(f)
            assert np.array_equal(got, (x / f(top)).astype(f)), (other, top)


# ----------------------------------------------------------------------------------------------------------
# the wrapper with stand-ins for tensors, streams and the library
# ----------------------------------------------------------------------------------------------------------

class FakeTensor:
    """What the wrapper asks of a CUDA tensor. `pool` is the stream whose memory it was allocated from."""

    def __init__(self, shape, dtype, env, pool=None):
        import math
        self.shape, self.dtype, self.env, self.pool, self.recorded = tuple(shape), dtype, env, pool, []
        self.n, self.is_cuda = math.prod(self.shape), True

    def _new(self, shape, dtype):
        t = FakeTensor([shape] if isinstance(shape, int) else shape, dtype, self.env, self.env.current)
        self.env.made.append(t)
        return t

    def new_empty(self, shape, dtype=None):
        return self._new(shape, dtype or self.dtype)

    def stride(self):
        strides, n = [], 1
        for d in reversed(self.shape):
            strides.append(n)
            n *= d
        return tuple(reversed(strides))

    def numel(self):
        return self.n

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def get_device(self):
        return 0

    def data_ptr(self):
        return FAKE

    def record_stream(self, stream):
        self.recorded.append(stream)


class FakeStream:
    def __init__(self, device_index=0):
        self.device_index, self.cuda_stream = device_index, 0x1234


class FakeEnv:
    """The wrapper on device 0 with torch's current stream and the library's entry points replaced."""

    def __init__(self, monkeypatch, max_new=40):
        import contextlib

        import torch
        from example_matmul_metal4_b200.kv_cache import KVCacheBatch, KVCacheDimensions, KVCachePlan
        self.made, self.calls, self.main = [], [], FakeStream()
        self.current = self.main

        @contextlib.contextmanager
        def on(stream):
            kept, self.current = self.current, stream
            yield
            self.current = kept

        monkeypatch.setattr(torch.cuda, "stream", on)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: self.current)
        monkeypatch.setattr(_lib, "stream_handle", lambda stream=None: None)
        i32 = torch.int32
        self.plan = KVCachePlan(KVCacheDimensions(7, 64, 8, 2, 128))
        self.batch = KVCacheBatch(FakeTensor((3, 4), i32, self), FakeTensor((3,), i32, self),
                                  FakeTensor((4,), i32, self), 5, max_new)
        real, env = self.plan._L, self

        class Library:
            def __getattr__(self, name):
                if name in ("mm4_kv_cache_append", "mm4_kv_cache_read", "mm4_kv_cache_attention"):
                    return lambda *a: env.calls.append((name, a)) or 0
                return getattr(real, name)

        self.plan._L, self.plan._device = Library(), lambda: 0
        self.plan._empty_like = lambda t: t._new(t.shape, t.dtype)
        self.cache = FakeTensor((7, self.plan.pageBytes), torch.uint8, self)
        self.Q = FakeTensor((5, 8, 128), torch.float16, self)
        self.K = FakeTensor((5, 2, 128), torch.float16, self)


def test_tensors_that_a_call_makes_come_from_the_memory_of_its_stream(monkeypatch):
    """A block of the current stream's pool may still be written by pending work of that stream, which a kernel on
    another stream does not wait for. What is returned is kept from reuse until the caller's stream is done with it."""
    env = FakeEnv(monkeypatch)
    side = FakeStream()
    for stream in (None, side):
        env.made.clear()
        O = env.plan.attention(env.Q, env.cache, env.batch, stream=stream)
        K, V = env.plan.read(env.cache, env.batch, stream=stream)
        assert len(env.made) == 4 and env.current is env.main  # O, workspace, K, V
        for t in env.made:
            assert t.pool is (env.main if stream is None else side)
        for t in (O, K, V):
            assert t.recorded == ([] if stream is None else [env.main])
        assert O.shape == (5, 8, 128) and K.shape == V.shape == (5, 2, 128)
    assert len(env.calls) == 4


def test_a_stream_of_another_device_is_refused(monkeypatch):
    env = FakeEnv(monkeypatch)
    for call in (lambda s: env.plan.append(env.K, env.K, env.cache, env.batch, stream=s),
                 lambda s: env.plan.read(env.cache, env.batch, stream=s),
                 lambda s: env.plan.attention(env.Q, env.cache, env.batch, stream=s)):
        with pytest.raises(ValueError, match="device 1"):
            call(FakeStream(1))
        call(FakeStream(0))
    assert len(env.calls) == 3


def test_attributes_of_a_batch_are_fixed(monkeypatch):
    """Another tensor in place of a batch's would leave the old address in the descriptor and drop its memory."""
    import torch
    env = FakeEnv(monkeypatch)
    for name in ("pageTable", "lengths", "offsets", "tokens", "maxNew", "sequences", "device", "desc"):
        kept = getattr(env.batch, name)
        with pytest.raises(AttributeError, match="fixed"):
            setattr(env.batch, name, FakeTensor((3,), torch.int32, env))
        assert getattr(env.batch, name) is kept
    env.plan.append(env.K, env.K, env.cache, env.batch)
    assert len(env.calls) == 1


def test_sizes_beyond_the_descriptors_are_refused(monkeypatch):
    """Sizes that would arrive as others, cut to 32 (pages: 64) bits."""
    import torch
    from example_matmul_metal4_b200.kv_cache import KVCacheBatch, KVCacheDimensions, KVCachePlan
    good = dict(pages=4, pageSize=64, Hq=8, Hk=2, K=128, bits=4)
    KVCachePlan(KVCacheDimensions(**good))
    for name, value in good.items():
        with pytest.raises(ValueError, match=name):
            KVCachePlan(KVCacheDimensions(**{**good, name: value + (1 << (64 if name == "pages" else 32))}))
    env = FakeEnv(monkeypatch)
    tensors = (FakeTensor((3, 4), torch.int32, env), FakeTensor((3,), torch.int32, env), FakeTensor((4,), torch.int32, env))
    for sizes in ((5 + (1 << 32), 2), (5, 2 + (1 << 32)), (5, 1 << 31)):
        with pytest.raises(ValueError, match="out of range"):
            KVCacheBatch(*tensors, *sizes)


@pytest.mark.parametrize("scale,used", [(None, 1 / 128 ** 0.5), (0, 1 / 128 ** 0.5), (-2.0, 1 / 128 ** 0.5), (1e-60, 1 / 128 ** 0.5),
                                        (0.25, 0.25), (1, 1.0)])
def test_scale_of_a_plan_is_the_one_that_its_kernels_use(scale, used):
    """A scale of 0 or less (in fp32) selects 1 / sqrt(head_dim)."""
    from example_matmul_metal4_b200.kv_cache import KVCacheDimensions, KVCachePlan
    assert KVCachePlan(KVCacheDimensions(4, 64, 8, 2, 128), scale=scale).scale == used
    for bad in (float("nan"), float("inf"), 1e300):
        with pytest.raises(_lib.MM4Error):
            KVCachePlan(KVCacheDimensions(4, 64, 8, 2, 128), scale=bad)


@pytest.mark.parametrize("max_new", [2, 13])
def test_attention_in_place_of_its_queries_is_refused(max_new):
    L = _lib.lib()
    rc, h = _plan()
    assert rc == 0
    assert L.mm4_kv_cache_attention(h, ctypes.byref(_batch(max_new=max_new)), FAKE, 1024, FAKE, FAKE, 1024, None, FAKE,
                                    1 << 40, None) == INVALID
    assert b"must not be Q" in L.mm4_last_error()
    L.mm4_kv_cache_plan_destroy(h)


def test_scale_whose_product_with_log2_e_is_infinite_is_refused():
    for scale, want in ((2.0 ** 127, 0), (2.3e38, 0), (2.4e38, UNSUPPORTED), (3.4e38, UNSUPPORTED), (-3.4e38, 0)):
        rc, h = _plan(scale=scale)
        assert rc == want, scale
        _lib.lib().mm4_kv_cache_plan_destroy(h)
