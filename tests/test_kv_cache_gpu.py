"""The key / value cache operators on the GPU against their float64 restatement (kv_cache_ref.py): written
bytes, read-back values and attention, at the lengths, heads, pages and masks where they can go wrong."""
import numpy as np
import pytest

import kv_cache_ref as ref
from example_matmul_metal4_b200 import data, sync_check
from example_matmul_metal4_b200._lib import MM4_ERR_INVALID, MM4Error
from example_matmul_metal4_b200.attention import MM4_ATTN_BSHD, AttentionDimensions, AttentionPlan
from example_matmul_metal4_b200.kv_cache import KVCacheBatch, KVCacheDimensions, KVCachePlan

pytestmark = pytest.mark.gpu


def _table(lengths, page, pages, seed, width=None):
    """A page table whose sequences use distinct pages of the pool in a random order; unused entries point
    outside the pool (they must not be read)."""
    rng = np.random.default_rng(seed)
    order = rng.permutation(pages)
    width = width or max(1, max((ln + page - 1) // page for ln in lengths))
    table = np.full((len(lengths), width), 2 ** 30, dtype=np.int32)
    at = 0
    for b, ln in enumerate(lengths):
        n = (ln + page - 1) // page
        table[b, :n] = order[at:at + n]
        at += n
    assert at <= pages
    return table


def _pages_for(lengths, page):
    return sum((ln + page - 1) // page for ln in lengths) + 2


class Setup:
    """A filled cache and a batch, on the host (bytes) and on the device."""

    def __init__(self, dev, lengths, new, Hq, Hk, D=128, bits=4, page=64, causal=True, seed=1, pad=0, scale=None,
                 maxNew=None, k_map=lambda k: k):
        import torch
        self.lengths, self.new, self.Hq, self.Hk, self.D, self.bits, self.page = lengths, new, Hq, Hk, D, bits, page
        self.causal, self.pad = causal, pad
        pages = _pages_for(lengths, page)
        self.plan = KVCachePlan(KVCacheDimensions(pages, page, Hq, Hk, D, bits), causal=causal, scale=scale)
        self.table = _table(lengths, page, pages, seed)
        self.offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.tokens = int(self.offsets[-1]) + pad
        # unused rows hold bytes whose scales and zeros are NaN: they must not reach any result
        self.host = np.full((pages, Hk, 2, page, ref.row_bytes(D, bits)), 0xFF, dtype=np.uint8)
        self.K, self.V = [], []
        for b, ln in enumerate(lengths):
            k = k_map(data.normal((ln, Hk, D), 1.0, seed, 10 + 2 * b).astype(np.float32))
            v = data.normal((ln, Hk, D), 1.0, seed, 11 + 2 * b)
            rows = [ref.pack(k.astype(np.float16), bits), ref.pack(v, bits)] if ln else None
            if ln:
                pos = np.arange(ln)
                for kv in (0, 1):
                    self.host[self.table[b, pos // page], :, kv, pos % page] = rows[kv]
            self.K.append(ref.unpack(rows[0], D, bits) if ln else np.zeros((0, Hk, D), np.float16))
            self.V.append(ref.unpack(rows[1], D, bits) if ln else np.zeros((0, Hk, D), np.float16))
        self.Q = data.normal((max(1, self.tokens), Hq, D), 1.0, seed, 5)[:self.tokens]
        self.dev = dev
        self.cache = torch.from_numpy(self.host.reshape(pages, -1)).to(dev)
        self.batch = KVCacheBatch(torch.from_numpy(self.table).to(dev),
                                  torch.tensor(lengths, dtype=torch.int32, device=dev),
                                  torch.from_numpy(self.offsets).to(dev), self.tokens,
                                  max(new) if maxNew is None else maxNew)

    def check(self, O, lse=None, sequences=None):
        O = O.double().cpu().numpy()
        lse = None if lse is None else lse.double().cpu().numpy()
        for b in range(len(self.lengths)) if sequences is None else sequences:
            r = slice(self.offsets[b], self.offsets[b + 1])
            eO, eL, tO, tL = ref.attention(self.Q[r], self.K[b], self.V[b], self.new[b], self.causal, self.plan.scale)
            off = np.abs(O[r] - eO) / np.maximum(tO, 2.0 ** -25)
            assert off.size == 0 or off.max() <= 1.0, (b, off.max(), np.unravel_index(off.argmax(), off.shape))
            if lse is not None:
                empty = np.isneginf(eL)
                assert np.array_equal(empty, np.isneginf(lse[r])), b
                d = np.abs(np.where(empty, 0, lse[r]) - np.where(empty, 0, eL))
                assert (d <= tL).all(), (b, (d - tL).max())

    def attend(self, want_lse=True, **kw):
        import torch
        Q = torch.from_numpy(np.ascontiguousarray(self.Q)).to(self.dev)
        lse = torch.full((self.tokens, self.Hq), 7.0, device=self.dev) if want_lse else None
        O = self.plan.attention(Q, self.cache, self.batch, lse=lse, **kw)
        sync_check()
        return O, lse


# ----------------------------------------------------------------------------------------------------------
# write and read back
# ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("D,Hk,page", [(128, 8, 64), (64, 1, 16), (128, 1, 256), (64, 5, 32), (128, 3, 128)])
def test_append_writes_the_defined_bytes_and_nothing_else(cuda, D, Hk, page, bits):
    """Ragged sequences whose new tokens start inside a page, end inside one and cross pages; strided K and V;
    padding rows behind the last sequence. Every byte of the cache is compared."""
    import torch
    lengths, new, pad = [300, 17, 1, 64, 33], [290, 5, 1, 64, 0], 3
    pages = _pages_for(lengths, page)
    plan = KVCachePlan(KVCacheDimensions(pages, page, Hk, Hk, D, bits))
    table = _table(lengths, page, pages, 3)
    offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    tokens = int(offsets[-1]) + pad
    K = data.normal((tokens, Hk, D), 2.0, 4, 0)
    V = data.normal((tokens, Hk, D), 0.5, 4, 1)
    host = np.full((pages, Hk, 2, page, ref.row_bytes(D, bits)), 0xA5, dtype=np.uint8)
    cache = torch.from_numpy(host.reshape(pages, -1).copy()).to(cuda)
    for b, (ln, n) in enumerate(zip(lengths, new)):
        pos = np.arange(ln - n, ln)
        r = slice(offsets[b], offsets[b + 1])
        host[table[b, pos // page], :, 0, pos % page] = ref.pack(K[r], bits)
        host[table[b, pos // page], :, 1, pos % page] = ref.pack(V[r], bits)
    fused = torch.zeros(tokens, 2 * Hk * D + 8, dtype=torch.float16, device=cuda)
    fused[:, :Hk * D] = torch.from_numpy(K.reshape(tokens, -1)).to(cuda)
    fused[:, Hk * D:2 * Hk * D] = torch.from_numpy(V.reshape(tokens, -1)).to(cuda)
    tK, tV = (fused[:, i * Hk * D:(i + 1) * Hk * D].view(tokens, Hk, D) for i in (0, 1))
    batch = KVCacheBatch(torch.from_numpy(table).to(cuda), torch.tensor(lengths, dtype=torch.int32, device=cuda),
                         torch.from_numpy(offsets).to(cuda), tokens, max(new))
    plan.append(tK, tV, cache, batch)
    sync_check()
    assert np.array_equal(cache.cpu().numpy().reshape(host.shape), host)
    # and back, into strided outputs whose padding rows stay as they were
    out = torch.full((tokens, 2 * Hk * D + 8), -3.0, dtype=torch.float16, device=cuda)
    oK, oV = (out[:, i * Hk * D:(i + 1) * Hk * D].view(tokens, Hk, D) for i in (0, 1))
    plan.read(cache, batch, K=oK, V=oV)
    sync_check()
    used = int(offsets[-1])
    assert np.array_equal(oK[:used].cpu().numpy(), ref.unpack(ref.pack(K[:used], bits), D, bits))
    assert np.array_equal(oV[:used].cpu().numpy(), ref.unpack(ref.pack(V[:used], bits), D, bits))
    assert (out[used:] == -3.0).all() and (out[:, 2 * Hk * D:] == -3.0).all()


@pytest.mark.parametrize("tokens,Hk,D,bits,per_warp", [(9501, 5, 128, 4, 2), (9600, 5, 128, 8, 2), (30001, 1, 128, 8, 3),
                                                       (47403, 3, 64, 8, 5), (76003, 3, 64, 4, 8)])
def test_append_and_read_of_several_tokens_a_warp(cuda, tokens, Hk, D, bits, per_warp):
    """Calls large enough for a warp to take several tokens, which cross sequences of every length, empty ones and
    rows before position 0 among them; padding at both ends, a last warp with fewer tokens, strides of their own for K
    and V. Every byte of the cache and every row is compared."""
    import torch
    sms = torch.cuda.get_device_properties(cuda).multi_processor_count
    parts = (2 * Hk * D // 8 + 127) // 128
    assert max(1, min(8, tokens * parts // (64 * sms))) == per_warp
    rng = np.random.default_rng(tokens)
    page, first, last = 32, 5, tokens - 3
    cut = np.unique(np.concatenate([[first, last], first + 1 + rng.integers(0, last - first - 1, 300),
                                    first + np.arange(1, 40)]))
    new = np.diff(cut)
    new = np.insert(new, [0, 17, 17, len(new)], 0)                    # sequences without rows
    offsets = (first + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)
    assert offsets[-1] == last
    lengths = (new + rng.integers(0, 50, len(new))).astype(np.int32)
    lengths[::9] = np.maximum(0, new[::9] - 4)                        # rows before position 0
    used = (lengths + page - 1) // page
    pages, table = int(used.sum()) + 2, np.full((len(new), int(used.max())), 2 ** 30, np.int32)
    order, at = rng.permutation(pages), 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    K, V = data.normal((tokens, Hk, D), 1.0, tokens, 0), data.normal((tokens, Hk, D), 2.0, tokens, 1)
    packed = [ref.pack(x, bits) for x in (K, V)]
    values = [ref.unpack(x, D, bits) for x in packed]
    t = np.arange(first, last)
    b = np.searchsorted(offsets, t, side="right") - 1
    pos = lengths[b] - (offsets[b + 1] - t)
    placed = pos >= 0
    t, b, pos = t[placed], b[placed], pos[placed]
    host = np.full((pages, Hk, 2, page, ref.row_bytes(D, bits)), 0xA5, dtype=np.uint8)
    cache = torch.from_numpy(host.reshape(pages, -1).copy()).to(cuda)
    for kv in (0, 1):
        host[table[b, pos // page], :, kv, pos % page] = packed[kv][t]
    width = Hk * D
    strided = [torch.full((tokens, width + extra), -3.0, dtype=torch.float16, device=cuda) for extra in (8, 24)]
    k, v = (x[:, :width].unflatten(1, (Hk, D)) for x in strided)
    k.copy_(torch.from_numpy(K))
    v.copy_(torch.from_numpy(V))
    i32 = dict(dtype=torch.int32, device=cuda)
    batch = KVCacheBatch(torch.from_numpy(table).to(cuda), torch.tensor(lengths, **i32), torch.tensor(offsets, **i32),
                         tokens, int(new.max()))
    plan = KVCachePlan(KVCacheDimensions(pages, page, Hk, Hk, D, bits))
    plan.append(k, v, cache, batch)
    sync_check()
    assert np.array_equal(cache.cpu().numpy().reshape(host.shape), host)
    for x in strided:
        x.fill_(-3.0)
    plan.read(cache, batch, K=k, V=v)
    sync_check()
    for kv, x in enumerate(strided):
        want = np.full(x.shape, -3.0, np.float16)
        want[t, :width] = values[kv][t].reshape(len(t), width)
        assert np.array_equal(x.cpu().numpy(), want)


@pytest.mark.parametrize("bits", [4, 8])
def test_groups_at_the_edges_of_fp16(cuda, bits):
    """Constant groups, zeros of both signs, NaN and infinities, the widest range, subnormals, a range of one
    smallest step, and values that land half-way between codes."""
    import torch
    top = 2 ** bits - 1
    g = np.zeros((16, 32), dtype=np.float16)
    g[0] = 1.5
    g[1, ::2] = -0.0
    g[2, :3] = [np.nan, np.inf, -np.inf]
    g[3] = np.where(np.arange(32) % 2, 65504, -65504)
    g[4] = np.arange(32) * 2.0 ** -24
    g[5, 7] = 2.0 ** -24
    g[6] = np.minimum(np.arange(32), top) * 0.5 + 0.25 * (np.arange(32) % 2)   # halves of the step 0.5 * k
    g[7] = np.nan
    g[8] = np.inf
    g[9] = -np.inf
    g[10] = np.linspace(-65504, 65504, 32)
    g[11] = 1024 + np.arange(32)
    g[12] = np.linspace(-1, 1, 32) * 2.0 ** -14
    g[13, 31] = 65504
    g[14, 0] = -65504
    g[15] = np.arange(32) / top
    x = g.reshape(4, 1, 128)
    plan = KVCachePlan(KVCacheDimensions(1, 16, 1, 1, 128, bits))
    cache = plan.allocate(cuda)
    t = torch.from_numpy(x).to(cuda)
    batch = KVCacheBatch(torch.zeros(1, 1, dtype=torch.int32, device=cuda),
                         torch.tensor([4], dtype=torch.int32, device=cuda),
                         torch.tensor([0, 4], dtype=torch.int32, device=cuda), 4, 4)
    plan.append(t, t.flip(0), cache, batch)
    K, V = plan.read(cache, batch)
    sync_check()
    want = ref.unpack(ref.pack(x, bits), 128, bits)
    got = K.cpu().numpy()
    assert np.isfinite(got).all()
    assert np.array_equal(got, want)
    assert np.array_equal(V.cpu().numpy(), want[::-1])
    # The error itself: half a step, plus what cutting the scale loses at the top code (2^-10 of top * scale, or
    # top * 2^-24 where scales are subnormal), plus fp16 rounding of the value.
    clean = np.clip(np.nan_to_num(x.astype(np.float64), nan=0.0), -65504, 65504)
    v = clean.reshape(16, 32)
    rng_ = v.max(1) - v.min(1)
    bound = rng_ / top * 0.5 + rng_ * 2.0 ** -10 + top * 2.0 ** -24
    err = np.abs(got.reshape(16, 32).astype(np.float64) - v)
    assert (err <= bound[:, None] + 2.0 ** -11 * np.abs(v) + 2.0 ** -25).all()


# ----------------------------------------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 255, 513, 1000])
def test_single_token_lengths(cuda, length, bits, D):
    s = Setup(cuda, [length], [1], 8, 2, D=D, bits=bits)
    s.check(*s.attend())


@pytest.mark.parametrize("D,bits", [(128, 4), (64, 8)])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (8, 8), (6, 2), (8, 1), (10, 5), (16, 1), (7, 1), (24, 2), (40, 1)])
def test_head_groups(cuda, Hq, Hk, D, bits):
    s = Setup(cuda, [333, 40], [1, 1], Hq, Hk, D=D, bits=bits, page=32)
    s.check(*s.attend())


@pytest.mark.parametrize("D,bits,page", [(128, 4, 16), (128, 8, 128), (64, 4, 256), (64, 8, 32)])
@pytest.mark.parametrize("new", [2, 3, 5, 16, 17, 64, 65, 130, 200])
@pytest.mark.parametrize("causal", [True, False])
def test_rows_of_one_sequence(cuda, new, causal, D, bits, page):
    """From two proposed tokens to prompt chunks, as the last rows of longer sequences and as whole ones."""
    s = Setup(cuda, [new + 300, new], [new, new], 4, 2, D=D, bits=bits, page=page, causal=causal)
    s.check(*s.attend())


@pytest.mark.parametrize("D,bits", [(128, 4), (64, 4), (128, 8), (64, 8)])
@pytest.mark.parametrize("new", [1, 4, 150])
def test_ragged_batches(cuda, new, D, bits):
    """Many sequences of lengths from one token to over a thousand, some with fewer rows, one with none."""
    rng = np.random.default_rng(new)
    lengths = [1, 1031, 2, 500, 64, 65, 127, 700, 33, 8, 1024, 90]
    n = [int(min(ln, rng.integers(1, new + 1))) for ln in lengths]
    n[3] = 0
    n[1] = new
    s = Setup(cuda, lengths, n, 8, 4, D=D, bits=bits, page=32, maxNew=new)
    s.check(*s.attend())


def test_prompt_over_several_row_blocks(cuda):
    """A prompt of more rows than one block of the kernel holds, grouped heads, with and without a cached prefix."""
    s = Setup(cuda, [700, 911], [700, 333], 6, 2, page=64)
    s.check(*s.attend())


@pytest.mark.parametrize("new,maxNew", [(1, 1), (9, 9), (300, 300)])
def test_rows_that_attend_to_nothing(cuda, new, maxNew):
    """Length 0, and more rows than the length: O = 0 and lse = -inf for the rows before position 0; padding rows
    of O and lse are left as they were."""
    import torch
    lengths, rows = [0, 5, 40, 3], [1, new, 1, 0]
    for causal in (True, False):
        s = Setup(cuda, lengths, rows, 4, 4, page=16, causal=causal, pad=2, maxNew=maxNew)
        O = torch.full((s.tokens, 4, 128), 9.0, dtype=torch.float16, device=cuda)
        got, lse = s.attend(O=O)
        assert got is O
        s.check(got, lse)
        assert (got[s.tokens - 2:] == 9.0).all() and (lse[s.tokens - 2:] == 7.0).all()
        if causal and new > 5:
            assert (got[1:1 + new - 5] == 0).all()


@pytest.mark.parametrize("new,length", [(1, 0), (9, 5), (60, 30), (300, 40)])
@pytest.mark.parametrize("bits", [4, 8])
def test_rows_that_attend_to_nothing_at_head_dim_64(cuda, bits, new, length):
    """O = 0 and lse = -inf exactly, where part of the exponentials comes from a polynomial that never gives 0."""
    s = Setup(cuda, [length, 700, length], [new, new, new], 4, 2, D=64, bits=bits, page=16)
    O, lse = s.attend()
    s.check(O, lse)
    empty = new - min(new, length)
    assert (O[:empty] == 0).all() and (lse[:empty] == -float("inf")).all()


@pytest.mark.parametrize("new", [1, 12, 70])
def test_large_scores(cuda, new):
    """Keys that grow along the sequence and a large scale, so the running maximum moves far and often."""
    s = Setup(cuda, [900], [new], 4, 2, scale=0.5, k_map=lambda k: k * np.linspace(0.25, 3.0, len(k))[:, None, None])
    s.check(*s.attend())


@pytest.mark.parametrize("new", [1, 40])
def test_scores_far_below_zero(cuda, new):
    """Every score of every row lies far below zero: exponentials are taken against the row's own maximum."""
    s = Setup(cuda, [200], [new], 2, 2, D=64, scale=1.0, k_map=np.abs)
    s.Q = -np.abs(s.Q)
    s.check(*s.attend())


def _exact_scores(s, S, sequence=0):
    """(O, lse, tol_O, tol_lse) in float64 of the rows of one sequence whose scores before scaling, S [n][Hq][len], are
    exact in fp32. What kv_cache_ref.attention derives, with ds = 0, and: the exponent y = (s - max) scale log2 e has two
    roundings of its own and two of the factor, 2^-22 |y| in all, which shift p by as much (ln 2 < 1); a small P is off
    by 2^-32 of the row's largest, as P is 2^7 p and fp16's steps are 2^-24."""
    n, Hq, ln = S.shape
    V = s.V[sequence].astype(np.float64).repeat(Hq // s.Hk, 1)                       # [len][Hq][D]
    scale = float(np.float32(s.plan.scale))
    if s.causal:
        S = np.where(np.arange(ln)[None, None] > (ln - n + np.arange(n))[:, None, None], -np.inf, S)
    m = S.max(-1, keepdims=True)
    y = (S - m) * scale / np.log(2)
    p = np.exp2(y)
    total = p.sum(-1)
    off = np.where(p > 0, p * np.abs(np.maximum(y, -2000)) * 2.0 ** -22, 0)
    mean = lambda w, v: np.einsum("nhl,lhd->nhd", w, v) / total[..., None]            # noqa: E731
    O, a = mean(p, V), mean(p, np.abs(V))
    rest = 2.0 ** -11 + 2.0 ** -19 + (ln / 16 + 64) * 2.0 ** -23
    tol = a * rest + mean(off, np.abs(V)) + np.abs(O) * (off.sum(-1) / total)[..., None] \
        + np.abs(V).sum(0) * 2.0 ** -32 / total[..., None] + 2.0 ** -11 * np.abs(O) + 2.0 ** -25
    lse = m[..., 0] * scale + np.log(total)
    tol_lse = off.sum(-1) / total + 2.0 ** -20 + (ln / 16 + 64) * 2.0 ** -23 + 2.0 ** -22 * np.abs(lse) \
        + 2.0 ** -22 * np.abs(m[..., 0]) * scale
    return O, lse, tol, tol_lse


def _check_exact(s, S):
    O, lse = s.attend()
    eO, eL, tO, tL = _exact_scores(s, S)
    dO, dL = np.abs(O.double().cpu().numpy() - eO), np.abs(lse.double().cpu().numpy() - eL)
    assert (dO <= tO).all(), (np.nanmax(dO / tO), np.isnan(dO).sum())
    assert (dL <= tL).all(), (np.nanmax(dL / tL), np.isnan(dL).sum())


@pytest.mark.parametrize("D,bits", [(64, 8), (64, 4), (128, 4)])
@pytest.mark.parametrize("new,name", [(1, "few<8"), (10, "few<24"), (70, "many")])
@pytest.mark.parametrize("key", [64 * 3 + i for i in range(8)] + [0, 38, 63, 230])
def test_rows_that_one_key_dominates(cuda, key, new, name, D, bits):
    """One key has nearly all of a row's weight, at every position of a group of 8: lse is that key's score, and O its
    value, to fp32 and fp16 precision wherever the key lies."""
    c = np.zeros(300, np.float32)
    c[key] = 16
    s = Setup(cuda, [300], [new], 4, 2, D=D, bits=bits, scale=0.125, causal=False,
              k_map=lambda k: np.ones_like(k) * c[:, None, None])
    assert name in s.plan.attention_kernel_name(s.batch)
    s.Q = np.zeros((new, 4, D), np.float16)
    s.Q[:, :, D - 1] = np.resize(np.float16([10, 12, 16]), (new, 4))
    _check_exact(s, s.Q[:, :, D - 1].astype(np.float64)[..., None] * c)


@pytest.mark.parametrize("D,bits", [(128, 4), (64, 8)])
@pytest.mark.parametrize("new,length,Hq,Hk", [(1, 1900, 4, 2), (1, 20000, 4, 2), (6, 1500, 4, 2), (12, 400, 300, 150),
                                              (60, 300, 150, 150), (70, 2000, 4, 2)])
@pytest.mark.parametrize("below", [18.3, 25.4, 28.5])
def test_many_small_probabilities_add_up(cuda, below, new, length, Hq, Hk, D, bits):
    """One key with nearly all of a row's weight and values of 0, and thousands of keys 2^-18 to 2^-28 of it: O comes
    from those alone. Their share must not be lost to fp16."""
    import torch
    s = Setup(cuda, [length], [new], Hq, Hk, D=D, bits=bits, scale=np.log(2) / 64, causal=False)
    c, v = np.zeros(length, np.float32), np.ones(length, np.float32)
    c[length // 3], v[length // 3] = 64 * below, 0
    K, V = (torch.from_numpy(np.broadcast_to(x.astype(np.float16)[:, None, None], (length, Hk, D)).copy()).to(cuda)
            for x in (c, v))
    whole = KVCacheBatch(s.batch.pageTable, s.batch.lengths, torch.tensor([0, length], dtype=torch.int32, device=cuda),
                         length, length)
    s.plan.append(K, V, s.cache, whole)
    s.V = [V.cpu().numpy()]
    s.Q = np.zeros((new, Hq, D), np.float16)
    s.Q[:, :, 7] = 1
    _check_exact(s, np.broadcast_to(c.astype(np.float16).astype(np.float64), (new, Hq, length)))


@pytest.mark.parametrize("D,bits", [(128, 4), (64, 8), (64, 4), (128, 8)])
@pytest.mark.parametrize("new,length", [(1, 200), (1, 3000), (6, 150), (6, 2500), (12, 300), (70, 500), (200, 9000)])
@pytest.mark.parametrize("scale", [None, 4.0, 1e-3])
def test_scores_at_the_ends_of_fp16(cuda, scale, new, length, D, bits):
    """Q and K up to 65504 of either sign: scores of 2^32 and beyond, whose maximum still has to count exactly 1. K is
    constant in each row, so cached exactly, and Q has one element, so every score is one exact product."""
    rng = np.random.default_rng(new)
    c = rng.choice(np.float32([65504, 65472, 65504, 40000, 60000, 1.5, -3, -65504]), length)
    s = Setup(cuda, [length], [new], 4, 2, D=D, bits=bits, scale=scale, k_map=lambda k: np.ones_like(k) * c[:, None, None])
    q = np.resize(np.float16([65504, -65504, 1024, 1, -4096, 2.0 ** -10, 0, 65472, -65504]), (new, 4))
    s.Q = np.zeros((new, 4, D), np.float16)
    s.Q[:, :, 5] = q
    _check_exact(s, q.astype(np.float64)[..., None] * c.astype(np.float64))


@pytest.mark.parametrize("D,bits", [(128, 4), (64, 8)])
@pytest.mark.parametrize("new,length", [(1, 300), (3, 4000), (12, 300), (70, 500)])
@pytest.mark.parametrize("e", [126, 60, 20, -20, -60, -126])
def test_scales_at_the_ends_of_fp32(cuda, e, new, length, D, bits):
    """A row that sees one key only, rows with equal largest scores and rows of zeros, at scales of 2^126 to 2^-126; lse
    where fp32 holds it."""
    c = np.resize(np.float32([2, -3, 0.5, 2, 1.5, 0]), length)
    s = Setup(cuda, [length], [new], 4, 2, D=D, bits=bits, scale=2.0 ** e, k_map=lambda k: np.ones_like(k) * c[:, None, None])
    q = np.resize(np.float16([1, -1, 0, 2.0 ** -10, 300]), (new, 4))
    s.Q = np.zeros((new, 4, D), np.float16)
    s.Q[:, :, 9] = q
    O, lse = s.attend()
    eO, eL, tO, tL = _exact_scores(s, q.astype(np.float64)[..., None] * c.astype(np.float64))
    assert (np.abs(O.double().cpu().numpy() - eO) <= tO).all()
    got, held = lse.double().cpu().numpy(), np.abs(eL) < 1e38
    assert held.any() and (np.abs(got - eL) <= tL)[held].all()


@pytest.mark.parametrize("D,bits", [(128, 4), (64, 8)])
@pytest.mark.parametrize("new,length", [(1, 300), (1, 3000), (3, 4000), (12, 700), (70, 500)])
def test_rows_of_nan_and_infinities_stay_alone(cuda, new, length, D, bits):
    """A NaN or an infinity in a row of Q makes that row's results NaN, as in the formula. The other rows stay within
    their tolerance (not bit for bit: the many-row kernel takes the exponents of a large row's warp another way)."""
    s = Setup(cuda, [length, 77], [new, new], 8, 2, D=D, bits=bits, k_map=lambda k: np.abs(k) + 0.5)
    bad = [(0, 1, np.nan), (new - 1, 2, np.inf), (new, 7, np.nan), (2 * new - 1, 4, np.inf)]
    want = [ref.attention(s.Q[b * new:(b + 1) * new], s.K[b], s.V[b], new, True, s.plan.scale) for b in (0, 1)]
    eO, eL, tO, tL = (np.concatenate(x) for x in zip(*want))
    for r, h, x in bad:
        s.Q[r, h, D // 2] = x
    O, lse = (t.double().cpu().numpy() for t in s.attend())
    other = np.ones(lse.shape, bool)
    for r, h, _ in bad:
        assert np.isnan(O[r, h]).all() and np.isnan(lse[r, h]), (r, h)
        other[r, h] = False
    assert (np.abs(lse - eL) <= tL)[other].all() and (np.abs(O - eO) <= tO)[other].all()


@pytest.mark.parametrize("D,bits", [(128, 4), (64, 8)])
@pytest.mark.parametrize("e", [24, 27, 30])
@pytest.mark.parametrize("new,length", [(1, 900), (1, 5000), (12, 700), (70, 1500)])
def test_maximum_rises_by_single_steps_of_fp32(cuda, new, length, e, D, bits):
    """Scores 2^e plus 0, 1, 2, ... units in the last place, 5.3 in the log2 domain each: the margin by which the
    running maximum may be stale is close to what fp32 resolves, and P must not leave fp16."""
    unit = 2.0 ** (e - 23)
    for order in (np.arange(length), np.random.default_rng(e).permutation(length)):
        j = order % 2000
        s = Setup(cuda, [length], [new], 2, 2, D=D, bits=bits, scale=5.3 * np.log(2) / unit,
                  k_map=lambda k: np.where(np.arange(k.shape[-1]) < 32, 32768.0, 32.0 * j[:, None, None] + 0 * k))
        s.Q = np.zeros((new, 2, D), np.float16)
        s.Q[:, :, 3] = 2.0 ** (e - 15)      # times 2^15: 2^e
        s.Q[:, :, 40] = unit / 32           # times 32 j: j units
        _check_exact(s, np.broadcast_to(2.0 ** e + unit * j, (new, 2, length)).astype(np.float64))


@pytest.mark.parametrize("new", [1, 100])
def test_strided_queries_and_outputs(cuda, new):
    import torch
    s = Setup(cuda, [400, 222], [new, new], 8, 2, D=64)
    width = 8 * 64
    big = torch.zeros(s.tokens, 2 * width + 8, dtype=torch.float16, device=cuda)
    big[:, 8:8 + width] = torch.from_numpy(s.Q.reshape(s.tokens, -1)).to(cuda)
    out = torch.full((s.tokens, width + 16), 4.0, dtype=torch.float16, device=cuda)
    O = out[:, 8:8 + width].view(s.tokens, 8, 64)
    s.plan.attention(big[:, 8:8 + width].view(s.tokens, 8, 64), s.cache, s.batch, O=O)
    sync_check()
    s.check(O)
    assert (out[:, :8] == 4.0).all() and (out[:, 8 + width:] == 4.0).all()


@pytest.mark.parametrize("new,length", [(1, 20000), (6, 9000), (40, 5000)])
def test_long_axis_is_split_and_joined(cuda, new, length):
    s = Setup(cuda, [length], [new], 8, 2, page=128)
    s.check(*s.attend())


@pytest.mark.parametrize("new,maxNew", [(1, 1), (2, 2), (5, 5), (9, 12), (20, 24)])
def test_many_sequences_on_shared_pages(cuda, new, maxNew):
    """600 sequences that share one prefix's pages: every worker's range crosses heads and sequences of more than
    32 pages each, and page-table reads start over at each of them."""
    import torch
    Hq, Hk, D, page, longest = 8, 4, 64, 16, 800
    base = Setup(cuda, [longest], [new], Hq, Hk, D=D, page=page)
    B = 600
    lengths = [520 + (37 * b) % 281 for b in range(B)]
    offsets = np.arange(B + 1, dtype=np.int32) * new
    Q = data.normal((B * new, Hq, D), 1.0, 9, 0)
    batch = KVCacheBatch(torch.from_numpy(np.repeat(base.table, B, axis=0)).to(cuda),
                         torch.tensor(lengths, dtype=torch.int32, device=cuda), torch.from_numpy(offsets).to(cuda),
                         B * new, maxNew)
    O = base.plan.attention(torch.from_numpy(Q).to(cuda), base.cache, batch)
    sync_check()
    got = O.double().cpu().numpy()
    for b in range(0, B, 7):
        r = slice(b * new, (b + 1) * new)
        eO, _, tO, _ = ref.attention(Q[r], base.K[0][:lengths[b]], base.V[0][:lengths[b]], new, True, base.plan.scale)
        assert (np.abs(got[r] - eO) <= tO).all(), b


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("new,name", [(1, "few<8 rows, split>"), (2, "few<8 rows, split>"), (3, "few<16 rows, split>"),
                                      (4, "few<16 rows, split>"), (5, "few<24 rows, split>"), (11, "few<24 rows, split>"),
                                      (13, "many")])
def test_each_kernel_over_long_caches(cuda, new, name, bits, D):
    """More tokens than a unit of its own CTA takes: every row count, width and head_dim on ranges that are split, with
    lengths around the borders of tiles and pages, and a sequence of no row."""
    lengths, rows = [5003, 2049, 64, 31, 2500], [new, max(1, new - 1), new, 1, 0]
    s = Setup(cuda, lengths, rows, 8, 2, D=D, bits=bits, page=16, maxNew=new)
    assert name in s.plan.attention_kernel_name(s.batch)
    s.check(*s.attend())


def _check_rows(s, O, lse, b, rows):
    """Single rows of a causal sequence, each as the last token of what it sees."""
    for i in rows:
        r, seen = int(s.offsets[b]) + i, s.lengths[b] - s.new[b] + i + 1
        eO, eL, tO, tL = ref.attention(s.Q[r:r + 1], s.K[b][:seen], s.V[b][:seen], 1, True, s.plan.scale)
        assert (np.abs(O[r:r + 1].double().cpu().numpy() - eO) <= tO).all(), (b, i)
        assert (np.abs(lse[r:r + 1].double().cpu().numpy() - eL) <= tL).all(), (b, i)


@pytest.mark.parametrize("D,bits", [(128, 4), (64, 8)])
@pytest.mark.parametrize("sequences", [40, 70, 150])
def test_many_rows_of_many_sequences(cuda, sequences, D, bits):
    """More sequences than a warp has lanes, of up to 30 tokens with 4 heads each, some with none."""
    rng = np.random.default_rng(sequences)
    rows = rng.integers(1, 31, sequences)
    rows[[3, 33, sequences - 1]], rows[5] = 0, 30
    lengths = rows + rng.integers(0, 200, sequences)
    s = Setup(cuda, [int(x) for x in lengths], [int(x) for x in rows], 8, 2, D=D, bits=bits, page=32, maxNew=30)
    assert "many" in s.plan.attention_kernel_name(s.batch)
    s.check(*s.attend())


@pytest.mark.parametrize("D,bits", [(128, 4), (64, 8)])
@pytest.mark.parametrize("others", [0, 2, 45])
def test_more_row_blocks_than_a_warp_has_lanes(cuda, others, D, bits):
    """A prompt of 4200 tokens with 2 heads a key / value head: 33 blocks of 256 rows, alone, between fewer sequences
    than blocks and between more of them."""
    rng = np.random.default_rng(others)
    small = [int(x) for x in rng.integers(1, 60, others)]
    new = small[:others // 2] + [4200] + small[others // 2:]
    lengths = [n + int(rng.integers(0, 40)) for n in new]
    s = Setup(cuda, lengths, new, 4, 2, D=D, bits=bits)
    assert "many" in s.plan.attention_kernel_name(s.batch)
    O, lse = s.attend()
    big = others // 2
    s.check(O, lse, sequences=[b for b in range(others + 1) if b != big])
    _check_rows(s, O, lse, big, [0, 1, 63, 127, 128, 255, 256, 1000, 2047, 4096, 4150, 4199] +
                [int(x) for x in rng.integers(0, 4200, 30)])


@pytest.mark.parametrize("new", [1, 5, 200])
def test_repeated_calls_give_the_same_bits(cuda, new):
    import torch
    s = Setup(cuda, [3000, 1200, 77], [new, new, min(new, 77)], 8, 2)
    first, l0 = s.attend()
    for _ in range(5):
        again, l1 = s.attend()
        assert torch.equal(first, again) and torch.equal(l0, l1)


@pytest.mark.parametrize("D", [128, 64])
def test_agrees_with_the_dense_attention_on_the_values_read_back(cuda, D):
    """Non-causal attention over the cache against AttentionPlan on what `read` returns: both take the same fp16
    K and V, so they differ by the kernels' own rounding: twice the tolerance of one."""
    import torch
    B, S, H, Hk = 2, 320, 4, 2
    s = Setup(cuda, [S] * B, [S] * B, H, Hk, D=D, causal=False, page=64)
    K, V = s.plan.read(s.cache, s.batch)
    O, _ = s.attend()
    dense = AttentionPlan(AttentionDimensions(S, S, D, H, Hk), batch=B, layout=MM4_ATTN_BSHD)
    Q = torch.from_numpy(s.Q).to(cuda).view(B, S, H, D)
    want = dense.run(Q, K.view(B, S, Hk, D), V.view(B, S, Hk, D)).view(B * S, H, D)
    sync_check()
    s.check(O)
    tol = np.concatenate([ref.attention(s.Q[b * S:(b + 1) * S], s.K[b], s.V[b], S, False, s.plan.scale)[2]
                          for b in range(B)])
    assert (np.abs(O.double().cpu().numpy() - want.double().cpu().numpy()) <= 2 * tol).all()


# ----------------------------------------------------------------------------------------------------------
# together, as a program uses them
# ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("bits,D", [(4, 128), (8, 64)])
def test_prompt_then_tokens_one_by_one(cuda, bits, D):
    """A prompt is written and attended over, then single tokens, then three at once, on one cache, with the
    batch's tensors updated in place; every step against the definition on the values written so far."""
    import torch
    Hq, Hk, page, pages = 8, 2, 16, 40
    plan = KVCachePlan(KVCacheDimensions(pages, page, Hq, Hk, D, bits))
    cache = plan.allocate(cuda)
    table = np.random.default_rng(0).permutation(pages)[:36].reshape(2, 18).astype(np.int32)
    tt = torch.from_numpy(table).to(cuda)
    lengths = torch.zeros(2, dtype=torch.int32, device=cuda)
    held = [[np.zeros((0, Hk, D), np.float16)] * 2 for _ in range(2)]
    step = 0
    for new in ([200, 71], [1, 1], [1, 1], [1, 0], [3, 3], [1, 1]):
        step += 1
        offsets = torch.tensor([0, new[0], new[0] + new[1]], dtype=torch.int32, device=cuda)
        lengths += torch.tensor(new, dtype=torch.int32, device=cuda)
        tokens = sum(new)
        batch = KVCacheBatch(tt, lengths, offsets, tokens, max(new))
        K = data.normal((tokens, Hk, D), 1.0, 50 + step, 0)
        V = data.normal((tokens, Hk, D), 1.0, 50 + step, 1)
        Q = data.normal((tokens, Hq, D), 1.0, 50 + step, 2)
        plan.append(torch.from_numpy(K).to(cuda), torch.from_numpy(V).to(cuda), cache, batch)
        O = plan.attention(torch.from_numpy(Q).to(cuda), cache, batch)
        sync_check()
        got = O.double().cpu().numpy()
        at = 0
        for b in range(2):
            r = slice(at, at + new[b])
            at += new[b]
            for kv, x in ((0, K), (1, V)):
                held[b][kv] = np.concatenate([held[b][kv], ref.unpack(ref.pack(x[r], bits), D, bits)])
            eO, _, tO, _ = ref.attention(Q[r], held[b][0], held[b][1], new[b], True, plan.scale)
            assert (np.abs(got[r] - eO) <= tO).all(), (step, b)
    whole = [len(held[0][0]), len(held[1][0])]
    batch = KVCacheBatch(tt, lengths, torch.tensor([0, whole[0], sum(whole)], dtype=torch.int32, device=cuda),
                         sum(whole), max(whole))
    K, V = plan.read(cache, batch)
    sync_check()
    assert np.array_equal(K.cpu().numpy(), np.concatenate([held[0][0], held[1][0]]))
    assert np.array_equal(V.cpu().numpy(), np.concatenate([held[0][1], held[1][1]]))


def test_captured_step_replays_with_new_lengths(cuda):
    """append + attention of one token, captured once and replayed as the lengths grow; a second captured step
    of other sequences on the same plan, replayed in turn; both against the definition."""
    import torch
    Hq, Hk, D, page, pages = 8, 2, 128, 16, 64
    plan = KVCachePlan(KVCacheDimensions(pages, page, Hq, Hk, D, 4))
    states = []
    for g in range(2):
        cache = plan.allocate(cuda)
        table = torch.randperm(pages, device=cuda).to(torch.int32).view(2, 32)
        lengths = torch.tensor([100, 30 + g], dtype=torch.int32, device=cuda)
        offsets = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)
        whole = torch.tensor([0, 100, 130 + g], dtype=torch.int32, device=cuda)
        K0 = torch.from_numpy(data.normal((130 + g, Hk, D), 1.0, 60 + g, 0)).to(cuda)
        V0 = torch.from_numpy(data.normal((130 + g, Hk, D), 1.0, 60 + g, 1)).to(cuda)
        plan.append(K0, V0, cache, KVCacheBatch(table, lengths, whole, 130 + g, 100))
        batch = KVCacheBatch(table, lengths, offsets, 2, 1)
        K, V = torch.zeros(2, Hk, D, dtype=torch.float16, device=cuda), torch.zeros(2, Hk, D, dtype=torch.float16,
                                                                                 device=cuda)
        Q = torch.zeros(2, Hq, D, dtype=torch.float16, device=cuda)
        O = torch.zeros_like(Q)
        plan.attention(Q, cache, batch, O=O)  # warm-up
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.append(K, V, cache, batch)
            plan.attention(Q, cache, batch, O=O)
        k0, v0 = (ref.unpack(ref.pack(t.cpu().numpy(), 4), D, 4) for t in (K0, V0))
        held = [[k0[:100], v0[:100]], [k0[100:], v0[100:]]]
        states.append((graph, cache, lengths, K, V, Q, O, held, batch))  # the batch keeps its tensors alive
    for step in range(20):
        for g, (graph, cache, lengths, K, V, Q, O, held, _) in enumerate(states):
            lengths += 1
            for i, t in enumerate((K, V, Q)):
                t.copy_(torch.from_numpy(data.normal(tuple(t.shape), 1.0, 70 + step, 3 * g + i)))
            graph.replay()
            got = O.double().cpu().numpy()
            kn, vn = (ref.unpack(ref.pack(t.cpu().numpy(), 4), D, 4) for t in (K, V))
            for b in range(2):
                held[b][0] = np.concatenate([held[b][0], kn[b:b + 1]])
                held[b][1] = np.concatenate([held[b][1], vn[b:b + 1]])
                eO, _, tO, _ = ref.attention(Q[b:b + 1].cpu().numpy(), held[b][0], held[b][1], 1, True, plan.scale)
                assert (np.abs(got[b:b + 1] - eO) <= tO).all(), (step, g, b)
    sync_check()


FIRST_CALL_CAPTURED = """
import torch
from example_matmul_metal4_b200 import sync_check
from example_matmul_metal4_b200.kv_cache import KVCacheBatch, KVCacheDimensions, KVCachePlan
i32 = dict(dtype=torch.int32, device="cuda")
for new in (1, 100):
    plan = KVCachePlan(KVCacheDimensions(64, 64, 8, 2, 128))
    cache = plan.allocate("cuda")
    batch = KVCacheBatch(torch.arange(64, **i32).view(1, 64), torch.tensor([2500], **i32),
                         torch.tensor([0, new], **i32), new, new)
    K, V = (torch.randn(new, 2, 128, device="cuda").half() for _ in range(2))
    Q = torch.randn(new, 8, 128, device="cuda").half()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.append(K, V, cache, batch)
        O = plan.attention(Q, cache, batch)
        k, v = plan.read(cache, batch)
    graph.replay()
    graph.replay()
    sync_check()
    want = plan.attention(Q, cache, batch)
    sync_check()
    assert torch.equal(O, want) and torch.isfinite(O).all()
    assert (k.float() - K.float()).abs().max() < 0.5
print("captured")
"""


def test_first_calls_of_a_process_may_be_captured(cuda):
    """The library's first calls on a device, made inside a stream capture in a fresh process."""
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], cwd=Path(__file__).resolve().parents[1],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_wrapper_refusals(cuda):
    """Shapes, types, devices and layouts that the wrapper turns away before any launch."""
    import torch
    s = Setup(cuda, [100, 60], [2, 2], 4, 2, D=64)
    plan, cache, batch = s.plan, s.cache, s.batch
    Q = torch.from_numpy(s.Q).to(cuda)
    K = torch.zeros(4, 2, 64, dtype=torch.float16, device=cuda)
    bad_q = [Q.float(), Q[:3], Q.cpu(), torch.zeros(4, 4, 128, dtype=torch.float16, device=cuda)[:, :, ::2],
             torch.zeros(4, 64, 4, dtype=torch.float16, device=cuda).transpose(1, 2)]
    for q in bad_q:
        with pytest.raises(ValueError):
            plan.attention(q, cache, batch)
        with pytest.raises(ValueError):
            plan.attention(Q, cache, batch, O=q)
    for c in (cache.cpu(), cache[1:], cache.view(torch.int8), torch.cat([cache, cache], 1)[:, :plan.pageBytes]):
        for call in (lambda: plan.attention(Q, c, batch), lambda: plan.append(K, K, c, batch),
                     lambda: plan.read(c, batch)):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(ValueError):
        plan.append(K[:, :1], K, cache, batch)
    with pytest.raises(ValueError):
        plan.read(cache, batch, K=K)
    for lse in (torch.zeros(4, 4, device=cuda).half(), torch.zeros(4, 3, device=cuda), torch.zeros(4, 4),
                torch.zeros(4, 8, device=cuda)[:, ::2]):
        with pytest.raises(ValueError):
            plan.attention(Q, cache, batch, lse=lse)
    with pytest.raises(MM4Error):  # rows that are not 8 elements apart
        plan.attention(torch.zeros(4, 260, dtype=torch.float16, device=cuda)[:, :256].view(4, 4, 64), cache, batch)
    with pytest.raises(MM4Error):  # a base that is not 16-byte aligned
        plan.attention(torch.zeros(4 * 256 + 4, dtype=torch.float16, device=cuda)[4:].view(4, 4, 64), cache, batch)
    many = KVCacheBatch(batch.pageTable, batch.lengths, batch.offsets, 4, 40)
    small = torch.empty(plan.attention_workspace_bytes(many) - 16, dtype=torch.uint8, device=cuda)
    with pytest.raises(MM4Error):
        plan.attention(Q, cache, many, workspace=small)
    i32 = dict(dtype=torch.int32, device=cuda)
    t, ln, off = torch.zeros(2, 3, **i32), torch.zeros(2, **i32), torch.zeros(3, **i32)
    for args in ((t.long(), ln, off), (t[:1], ln, off), (t, ln[:1], off), (t, ln, off[:2]), (t.T, ln, off),
                 (t.view(-1), ln, off), (t, ln, off.cpu())):
        with pytest.raises(ValueError):
            KVCacheBatch(*args, 4, 2)
    with pytest.raises(ValueError):
        KVCacheBatch(t, ln, off, -1, 1)
    sync_check()


def test_given_workspace_and_empty_batches(cuda):
    """A workspace of the caller's with anything in it; batches without rows and without sequences do nothing."""
    import torch
    s = Setup(cuda, [3000], [20], 8, 2)
    ws = torch.full((s.plan.attention_workspace_bytes(s.batch) + 64,), 0xFF, dtype=torch.uint8, device=cuda)
    s.check(*s.attend(workspace=ws))
    i32 = dict(dtype=torch.int32, device=cuda)
    for seqs, tokens in ((0, 3), (2, 0), (0, 0)):
        b = KVCacheBatch(torch.zeros(seqs, 4, **i32), torch.zeros(seqs, **i32), torch.zeros(seqs + 1, **i32), tokens, 1)
        K = torch.ones(tokens, 2, 128, dtype=torch.float16, device=cuda)
        O = torch.ones(tokens, 8, 128, dtype=torch.float16, device=cuda)
        before = s.cache.clone()
        s.plan.append(K, K, s.cache, b)
        s.plan.read(s.cache, b, K=K, V=K.clone())
        s.plan.attention(O.clone(), s.cache, b, O=O)
        sync_check()
        assert (K == 1).all() and (O == 1).all() and torch.equal(before, s.cache)


def test_two_streams_at_once(cuda):
    """The same plan on two streams with work in flight on both; each call has a workspace of its own."""
    import torch
    a = Setup(cuda, [8000, 3001], [1, 1], 8, 2, seed=5)
    b = Setup(cuda, [5000], [3], 8, 2, seed=6)
    wa, wb = a.attend()[0], b.attend()[0]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    Qa, Qb = torch.from_numpy(a.Q).to(cuda), torch.from_numpy(b.Q).to(cuda)
    torch.cuda.synchronize()
    out = []
    for _ in range(20):
        out.append((a.plan.attention(Qa, a.cache, a.batch, stream=s1), b.plan.attention(Qb, b.cache, b.batch,
                                                                                        stream=s2)))
    torch.cuda.synchronize()
    for x, y in out:
        assert torch.equal(x, wa) and torch.equal(y, wb)


@pytest.mark.parametrize("new", [1, 40])
def test_memory_freed_on_the_current_stream_with_work_pending(cuda, new):
    """Blocks of the sizes of O, the workspace, K and V are freed on the current stream while it still has to write
    them; calls on another stream must not be given them."""
    import torch
    s = Setup(cuda, [3000], [new], 8, 2)
    Q = torch.from_numpy(s.Q).to(cuda)
    want = s.plan.attention(Q, s.cache, s.batch)
    K, V = s.plan.read(s.cache, s.batch)
    nbytes = s.plan.attention_workspace_bytes(s.batch)
    assert nbytes > 0
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        held = [torch.empty_like(t) for t in (want, K, V) for _ in range(3)]
        held += [torch.empty(nbytes, dtype=torch.uint8, device=cuda) for _ in range(3)]
        torch.cuda._sleep(20_000_000)  # about 10 ms
        for t in held:
            t.fill_(77)
        del held, t
        O = s.plan.attention(Q, s.cache, s.batch, stream=side)
        k, v = s.plan.read(s.cache, s.batch, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(O, want) and torch.equal(k, K) and torch.equal(v, V)


def test_cache_offsets_past_32_bits(cuda):
    """A pool of over 5 GB whose used pages lie at its end."""
    import torch
    page, Hk, D = 256, 16, 128
    page_bytes = Hk * 2 * page * ref.row_bytes(D, 4)
    pages = (5 << 30) // page_bytes
    plan = KVCachePlan(KVCacheDimensions(pages, page, Hk, Hk, D, 4))
    assert plan.cacheBytes > 1 << 32
    cache = plan.allocate(cuda)
    for new in (1, 200):
        ln = 300
        table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=cuda)
        lengths = torch.tensor([ln], dtype=torch.int32, device=cuda)
        K, V = data.normal((ln, Hk, D), 1.0, 80, 0), data.normal((ln, Hk, D), 1.0, 80, 1)
        Q = data.normal((new, Hk, D), 1.0, 80, 2)
        plan.append(torch.from_numpy(K).to(cuda), torch.from_numpy(V).to(cuda), cache,
                    KVCacheBatch(table, lengths, torch.tensor([0, ln], dtype=torch.int32, device=cuda), ln, ln))
        O = plan.attention(torch.from_numpy(Q).to(cuda), cache,
                           KVCacheBatch(table, lengths, torch.tensor([0, new], dtype=torch.int32, device=cuda), new,
                                        new))
        sync_check()
        k, v = (ref.unpack(ref.pack(x, 4), D, 4) for x in (K, V))
        eO, _, tO, _ = ref.attention(Q, k, v, new, True, plan.scale)
        assert (np.abs(O.double().cpu().numpy() - eO) <= tO).all()
    assert not cache[:pages - 2].any()


# ----------------------------------------------------------------------------------------------------------
# wrong batches: reported, contained
# ----------------------------------------------------------------------------------------------------------

def _reported(text):
    with pytest.raises(MM4Error, match=text) as e:
        sync_check()
    assert e.value.status == MM4_ERR_INVALID
    sync_check()  # reported once


@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("entry", [-1, 10 ** 6])
def test_a_page_outside_the_pool_is_reported_and_touches_no_other_sequence(cuda, entry, new):
    import torch
    s = Setup(cuda, [200, 150, 170], [new, new, new], 4, 2, page=32)
    s.batch.pageTable[1, 2] = entry
    Q = torch.from_numpy(s.Q).to(cuda)
    O = s.plan.attention(Q, s.cache, s.batch)
    _reported("page number")
    s.check(O, sequences=[0, 2])
    K, V = s.plan.read(s.cache, s.batch)
    if new > 1:  # rows 50 .. 149 reach the wrong entry, row 149 alone does not
        _reported("page number")
        s.plan.append(K, V, s.cache, s.batch)
        _reported("page number")
    sync_check()


@pytest.mark.parametrize("n", [1, 40, 7000])
@pytest.mark.parametrize("what", ["end beyond the rows", "start before the rows", "out of order", "negative length",
                                  "length beyond the table"])
def test_append_and_read_leave_out_wrong_sequences_and_report_them(cuda, what, n):
    """Three sequences of n rows each, one of them wrong: the others are written and read exactly, and no other byte
    changes. 21,000 rows take the form in which a warp has several tokens."""
    import torch
    Hk, D, page, bits = 2, 64, 64, 4
    lengths, offsets, wrong = [2 * n + 9, 2 * n + 30, 2 * n + 3], [0, n, 2 * n, 3 * n], []
    room = (max(lengths) + page - 1) // page
    table = np.random.default_rng(n).permutation(3 * room + 1)[:3 * room].reshape(3, room).astype(np.int32)
    told = list(lengths)
    if what == "end beyond the rows":
        offsets[3], wrong = 3 * n + 1, [2]
    elif what == "start before the rows":
        offsets[0], wrong = -1, [0]
    elif what == "out of order":
        offsets[1], offsets[2], wrong = 2 * n, n, [1]   # rows n .. 2 n - 1 are in sequences 0 and 2
    elif what == "negative length":
        told[1], wrong = -5, [1]
    else:
        told[1], wrong = room * page + 1, [1]
    plan = KVCachePlan(KVCacheDimensions(3 * room + 1, page, Hk, Hk, D, bits))
    K, V = data.normal((3 * n, Hk, D), 1.0, n, 0), data.normal((3 * n, Hk, D), 1.0, n, 1)
    packed = [ref.pack(x, bits) for x in (K, V)]
    values = [ref.unpack(x, D, bits) for x in packed]
    host = np.full((3 * room + 1, Hk, 2, page, ref.row_bytes(D, bits)), 0xA5, dtype=np.uint8)
    cache = torch.from_numpy(host.reshape(len(host), -1).copy()).to(cuda)
    batch = KVCacheBatch(torch.from_numpy(table).to(cuda), torch.tensor(told, dtype=torch.int32, device=cuda),
                         torch.tensor(offsets, dtype=torch.int32, device=cuda), 3 * n, n)
    plan.append(torch.from_numpy(K).to(cuda), torch.from_numpy(V).to(cuda), cache, batch)
    text = "length" if "length" in what else "offsets"
    _reported(text)
    free = np.zeros(host.shape[:1] + host.shape[3:4], dtype=bool)    # places of rows that two sequences hold
    read = np.zeros(3 * n, dtype=bool)
    either = np.zeros(3 * n, dtype=bool)
    if what == "out of order":
        either[n:2 * n] = True
    for b in range(3):
        if b in wrong:
            continue
        t = np.arange(max(0, offsets[b]), offsets[b + 1])
        pos = lengths[b] - (offsets[b + 1] - t)
        to, row = table[b, pos // page], pos % page
        for kv in (0, 1):
            host[to, :, kv, row] = packed[kv][t]
        free[to[either[t]], row[either[t]]] = True
        read[t] = True
    got = cache.cpu().numpy().reshape(host.shape)
    same = (got == host).all(axis=(1, 2, 4))
    assert same[~free].all() and (same | (got == 0xA5).all(axis=(1, 2, 4))).all()
    oK, oV = (torch.full((3 * n, Hk, D), -3.0, dtype=torch.float16, device=cuda) for _ in range(2))
    plan.read(torch.from_numpy(host.reshape(len(host), -1)).to(cuda), batch, K=oK, V=oV)
    _reported(text)
    for out, want in ((oK, values[0]), (oV, values[1])):
        out = out.cpu().numpy()
        assert np.array_equal(out[read & ~either], want[read & ~either])
        assert (out[~read] == -3.0).all()


def test_a_wrong_batch_is_reported_behind_a_run_out_wait(cuda):
    """A check reports one thing; what it does not report stays for the next."""
    from example_matmul_metal4_b200._lib import MM4_ERR_TIMEOUT, check, lib, stream_handle
    import torch
    s = Setup(cuda, [200], [1], 4, 2)
    s.batch.pageTable[0, 1] = -1
    s.plan.attention(torch.from_numpy(s.Q).to(cuda), s.cache, s.batch)
    check(lib().mm4_debug_wait_timeout(1_000_000, stream_handle()))  # a wait that runs out after 1 ms
    with pytest.raises(MM4Error) as e:
        sync_check()
    assert e.value.status == MM4_ERR_TIMEOUT
    _reported("page number")


@pytest.mark.parametrize("new", [1, 100])
def test_wrong_lengths_offsets_and_row_counts_are_reported(cuda, new):
    import torch
    s = Setup(cuda, [200, 150, 170], [new, new, new], 4, 2, page=32)
    Q = torch.from_numpy(s.Q).to(cuda)
    for value in (-5, 10 ** 6, 2 ** 31 - 1):
        s.batch.lengths[1] = value
        O = s.plan.attention(Q, s.cache, s.batch)
        with pytest.raises(MM4Error):  # a length too long also reaches the table's entries behind the sequence
            sync_check()
        sync_check()
        s.check(O, sequences=[0, 2])
    s.batch.lengths[1] = 150
    keep = s.batch.offsets.clone()
    for bad in ([0, new, 2 * new, 3 * new + 1], [0, new, 2 * new, -1]):
        s.batch.offsets.copy_(torch.tensor(bad, dtype=torch.int32))
        O = s.plan.attention(Q, s.cache, s.batch)
        _reported("offsets")
        s.check(O, sequences=[0, 1])
    s.batch.offsets.copy_(keep)
    few = KVCacheBatch(s.batch.pageTable, s.batch.lengths, torch.tensor([0, new, 2 * new, 3 * new], dtype=torch.int32,
                                                                       device=cuda), 3 * new, max(1, new - 1))
    if new > 1:
        s.plan.attention(Q, s.cache, few)
        _reported("max_new")
