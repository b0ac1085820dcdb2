"""Paged block memory on the GPU: block tables, append and shared-prefix attention
against the oracle (float64), at the sizes and masks where they can go wrong, and
run together as a serving loop would.

Tolerances of the attention.  With u = eps / 2 of the element type (half a step
of a rounding, relative), e = 2^-24 (fp32) and A = sum p |v| / sum p:
  output rounding                        u |o|
  weights rounded to 16 bits (not fp32)  u A
  a score's error, fp32 products and sums over d terms, the scale and the
    exponent's argument: s = (d + 8) e top, a factor (1 + s) on each weight,
    in numerator and denominator         2 s A
  exp2 and the sums of n weights         2 (n e + 2^-21) A
and for the log-sum-exp s + n e + 2^-21 + 2 e |lse|.  ``top`` is the largest
scale sum |q| |k| of the row."""
import math

import numpy as np
import pytest
import torch

from gfst_hmb_public_b200 import _native as nat
from gfst_hmb_public_b200 import paged
from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32


def _np(t):
    return t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _dev(x, dev, dtype=torch.int32):
    return torch.as_tensor(np.asarray(x).astype(np.int32)).to(dev, dtype)


# ---------------------------------------------------------------------------
# block tables
# ---------------------------------------------------------------------------
def _table_inputs(rng, B, W, L, hi_len, hi_new, ended, spare):
    lens = rng.integers(0, min(hi_len, W * L) + 1, B)
    new = np.minimum(rng.integers(0, hi_new + 1, B), W * L - lens)
    if ended:
        new[rng.random(B) < ended] = -1
    held = -(-lens // L)
    need = -(-(lens + np.maximum(new, 0)) // L)
    F = int(held.sum() + (need - held).sum()) + spare
    F = max(F, int(held.sum()) + 1)
    order = rng.permutation(F)
    tables, at = np.full((B, W), -1), 0
    for b in range(B):
        tables[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    head, ring = int(rng.integers(F)), np.full(F, -1)
    ring[(head + np.arange(F - at)) % F] = order[at:]
    return lens, new, tables, ring, np.array([head, F - at])


def _check_tables(dev, inputs, L, n_tokens, in_place):
    lens, new, tables, ring, state = inputs
    want = po.block_tables(lens, new, tables, ring, state, L, n_tokens)
    d = [_dev(x, dev) for x in inputs]
    got = paged.block_tables(d[0], d[1], d[2], d[3], d[4], block_len=L, n_tokens=n_tokens,
                             tables_out=d[2] if in_place else None)
    if not in_place:
        assert np.array_equal(_np(d[2]), tables)
    assert np.array_equal(_np(d[0]), lens) and np.array_equal(_np(d[4]), state)
    for name, g, w in zip(("tables", "lens", "cu_new", "slot_map", "free_state", "n_short"), got, want):
        assert np.array_equal(_np(g).reshape(-1), np.asarray(w).reshape(-1)), name
    assert np.array_equal(_np(d[3]), want[6])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B, W, L, hi_len, hi_new, ended, spare", [
    (1, 1, 1, 1, 1, 0, 0), (1, 5, 16, 0, 80, 0, 2), (3, 7, 16, 112, 5, 0.4, 1), (33, 9, 24, 100, 40, 0.2, 0),
    (256, 31, 64, 1500, 1, 0.05, 3), (257, 40, 16, 600, 0, 0, 1), (300, 12, 16, 150, 33, 1.0, 4),
    (1025, 17, 8, 120, 20, 0.1, 0), (5000, 5, 32, 160, 3, 0.3, 7),
])
def test_block_tables(cuda_device, B, W, L, hi_len, hi_new, ended, spare, in_place):
    rng = np.random.default_rng(B * 1000 + W)
    inputs = _table_inputs(rng, B, W, L, hi_len, hi_new, ended, spare)
    n = int(np.maximum(inputs[1], 0).sum())
    _check_tables(cuda_device, inputs, L, n + (B % 3), in_place)


def test_block_tables_most_requests(cuda_device):
    rng = np.random.default_rng(9)
    inputs = _table_inputs(rng, 16384, 3, 16, 40, 8, 0.1, 5)
    _check_tables(cuda_device, inputs, 16, int(np.maximum(inputs[1], 0).sum()), True)


@pytest.mark.parametrize("lack", [1, 2, 6])
def test_block_tables_short_of_blocks(cuda_device, lack):
    rng = np.random.default_rng(lack)
    lens, new, tables, ring, state = _table_inputs(rng, 12, 8, 16, 90, 30, 0.2, 0)
    state = np.array([state[0], max(0, state[1] - lack)])
    _check_tables(cuda_device, (lens, new, tables, ring, state), 16, int(np.maximum(new, 0).sum()), False)


@pytest.mark.parametrize("ring_short", [True, False])
def test_block_tables_short_step_in_place_changes_nothing(cuda_device, ring_short):
    # the ring is empty, or request 0 wants more than its table is wide
    lens, new, want = [3, 5, 8, 0], *(([2, 5, -1, 3], 1) if ring_short else ([14, 1, -1, 3], 2))
    tables = [[7, -1, -1], [2, 9, -1], [4, 1, -1], [-1, -1, -1]]
    ring, state = [0, 3, 5, 6, 8, 10, 11, -1, -1, -1], [0, 2 if ring_short else 7]
    d = [_dev(x, cuda_device) for x in (lens, new, tables, ring, state)]
    t = paged.block_tables(*d, block_len=4, n_tokens=30, tables_out=d[2])
    assert int(t.n_short) == want
    assert t.tables.tolist() == tables and d[3].tolist() == ring
    assert t.lens.tolist() == lens and t.free_state.tolist() == state
    assert (t.cu_new == 0).all() and (t.slot_map == -1).all()


def test_memory_takes_a_short_step_again(cuda_device):
    mem = paged.PagedMemory(6, 16, 1, 64, max_requests=3, max_blocks=5, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(0)
    make = lambda n, h: torch.randn((n, h, 64), generator=g, device=cuda_device).to(BF16)  # noqa: E731
    K = make(60, 1)
    mem.append(K, K, mem.extend(_dev([30, 30, 0], cuda_device), 60))
    before = [x.clone() for x in (mem.tables, mem.lens, mem.free_ring, mem.free_state, mem.pool_K)]
    new, more = _dev([3, 3, 17], cuda_device), make(23, 1)      # four blocks, two are free
    t = mem.extend(new, 23)
    mem.append(more, more, t)
    out, lse = mem.attend(make(23, 2), t, return_lse=True)
    assert int(t.n_short) == 2
    assert all(torch.equal(a, b) for a, b in
               zip(before, (mem.tables, mem.lens, mem.free_ring, mem.free_state, mem.pool_K)))
    assert (out == 0).all() and torch.isneginf(lse).all()
    t = mem.extend(_dev([0, -1, 0], cuda_device), 0)            # request 1 returns two
    assert int(t.n_short) == 0 and int(mem.free_state[1]) == 4
    t = mem.extend(_dev([3, 0, 17], cuda_device), 20)
    assert int(t.n_short) == 0 and mem.lens.tolist() == [33, 0, 17]
    assert int((mem.tables >= 0).sum()) == 5 and int(mem.free_state[1]) == 1


def test_block_tables_beyond_the_width(cuda_device):
    # request 1 wants 4 blocks of a table 2 wide; its tokens there have no slot
    inputs = (np.array([3, 5, 0]), np.array([2, 11, 4]), np.array([[7, -1], [2, 9], [-1, -1]]),
              np.array([0, 1, 3, 4, 5, 6, 8, 10, 11, -1, -1, -1]), np.array([0, 9]))
    _check_tables(cuda_device, inputs, 4, 17, False)


def test_block_tables_padding_and_fewer_tokens(cuda_device):
    rng = np.random.default_rng(5)
    inputs = _table_inputs(rng, 6, 8, 16, 60, 20, 0, 3)
    n = int(inputs[1].sum())
    _check_tables(cuda_device, inputs, 16, n + 37, False)
    _check_tables(cuda_device, inputs, 16, n - 5, False)
    _check_tables(cuda_device, inputs, 16, 0, False)


def test_block_tables_refuses(cuda_device):
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=cuda_device)  # noqa: E731
    ok = dict(block_len=16, n_tokens=2)
    with pytest.raises(RuntimeError, match="int32"):
        paged.block_tables(i(2).long(), i(2), i(2, 4), i(8), i(2), **ok)
    with pytest.raises(ValueError):
        paged.block_tables(i(2), i(3), i(2, 4), i(8), i(2), **ok)
    with pytest.raises(ValueError):
        paged.block_tables(i(2), i(2), i(8), i(8), i(2), **ok)
    with pytest.raises(RuntimeError):
        paged.block_tables(i(2), i(2), i(2, 4), i(16)[::2], i(2), **ok)
    flat = i(24)
    with pytest.raises(ValueError, match="overlaps"):
        paged.block_tables(i(2), i(2), flat[:8].view(2, 4), i(8), i(2), tables_out=flat[4:12].view(2, 4), **ok)
    with pytest.raises(RuntimeError, match="unsupported shape"):
        paged.block_tables(i(2), i(2), i(2, 4), i(8), i(2), block_len=0, n_tokens=2)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
@pytest.mark.parametrize("n, H, d, dv, L, F, strided", [
    (1, 1, 64, 64, 16, 2, False), (37, 3, 80, 16, 24, 5, False), (300, 8, 128, 128, 64, 9, True),
    (1000, 2, 256, 64, 16, 80, True),
])
def test_paged_append(cuda_device, dtype, n, H, d, dv, L, F, strided):
    g = torch.Generator(device=cuda_device).manual_seed(n)
    make = lambda *s: torch.randn(s, generator=g, device=cuda_device).to(dtype)  # noqa: E731
    pool_K, pool_V = make(F, H, L, d), make(F, H, L, dv)
    if strided:  # the keys and values of a fused projection
        both = make(n, 2 * H, d + dv)
        K, V = both[:, :H, :d], both[:, H:, d:]
        assert not K.is_contiguous()
    else:
        K, V = make(n, H, d), make(n, H, dv)
    slots = np.random.default_rng(n).permutation(F * L)[:n].astype(np.int64)
    slots[::7] = -1
    if n > 20:
        slots[3], slots[5] = F * L, 2 ** 31 - 1   # outside the pool: left out
    want_K, want_V = pool_K.clone(), pool_V.clone()
    for t, s in enumerate(slots):
        if 0 <= s < F * L:
            want_K[s // L, :, s % L] = K[t]
            want_V[s // L, :, s % L] = V[t]
    paged.paged_append(K, V, pool_K, pool_V, _dev(slots, cuda_device))
    assert torch.equal(pool_K, want_K) and torch.equal(pool_V, want_V)


def test_paged_append_misaligned_rows_are_copied(cuda_device):
    base = torch.randn(4 * 2 * 64 + 1, device=cuda_device).to(BF16)
    K = base[1:].view(4, 2, 64)                       # 2-byte aligned
    pool = torch.zeros((2, 2, 16, 64), dtype=BF16, device=cuda_device)
    pool_V = torch.zeros_like(pool)
    slots = _dev([3, 31, 0, 16], cuda_device)
    paged.paged_append(K, K, pool, pool_V, slots)
    for t, s in enumerate([3, 31, 0, 16]):
        assert torch.equal(pool[s // 16, :, s % 16], K[t]) and torch.equal(pool_V[s // 16, :, s % 16], K[t])


def test_paged_append_refuses(cuda_device):
    x = torch.zeros((3, 2, 64), dtype=BF16, device=cuda_device)
    pool = torch.zeros((4, 2, 16, 64), dtype=BF16, device=cuda_device)
    slots = torch.zeros(3, dtype=torch.int32, device=cuda_device)
    with pytest.raises(RuntimeError, match="mixed"):
        paged.paged_append(x.float(), x, pool, pool, slots)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        paged.paged_append(x.double(), x.double(), pool.double(), pool.double(), slots)
    with pytest.raises(RuntimeError, match="int32"):
        paged.paged_append(x, x, pool, pool, slots.long())
    with pytest.raises(ValueError):
        paged.paged_append(x[:, :1], x, pool, pool, slots)
    with pytest.raises(ValueError, match="contiguous"):
        paged.paged_append(x, x, pool[::2], pool[::2], slots)
    with pytest.raises(RuntimeError, match="backward"):
        paged.paged_append(x.clone().requires_grad_(), x, pool, pool, slots)
    odd = torch.zeros((3, 2, 60), dtype=BF16, device=cuda_device)
    odd_pool = torch.zeros((4, 2, 16, 60), dtype=BF16, device=cuda_device)
    with pytest.raises(RuntimeError, match="misaligned"):
        paged.paged_append(odd, odd, odd_pool, odd_pool, slots)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
class Setup:
    """A pool that is NaN wherever no query looks, and what is attended."""

    def __init__(self, dev, dtype, lens, new, prefix, H, G, d, L, *, dv=None, seed=0, spare=3, q_scale=1.5, hidden=None):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device=dev).manual_seed(seed)
        dv = d if dv is None else dv
        lens, new = np.asarray(lens), np.asarray(new)
        need, p_need = -(-lens // L), -(-prefix // L)
        F = int(need.sum()) + p_need + spare
        order = rng.permutation(F)
        W = max(1, int(need.max()))
        tables, at = np.full((len(lens), W), -1), p_need
        hidden = float("nan") if hidden is None else hidden
        self.pool_K = torch.full((F, H, L, d), hidden, dtype=dtype, device=dev)
        self.pool_V = torch.full((F, H, L, dv), hidden, dtype=dtype, device=dev)
        held = [(order[:p_need], prefix)]
        for b, k in enumerate(need):
            tables[b, :k] = order[at:at + k]
            held.append((tables[b], int(lens[b])))
            at += k
        for blocks, n in held:
            for p0 in range(0, n, L):
                m = min(L, n - p0)
                blk = int(blocks[p0 // L])
                self.pool_K[blk, :, :m] = torch.randn((H, m, d), generator=g, device=dev).to(dtype)
                self.pool_V[blk, :, :m] = torch.randn((H, m, dv), generator=g, device=dev).to(dtype)
        self.dtype, self.scale, self.L, self.prefix = dtype, 1.0 / math.sqrt(d), L, prefix
        self.np_tables, self.np_lens, self.np_cu = tables, lens, np.concatenate([[0], np.cumsum(new)])
        self.np_prefix = order[:p_need]
        self.tables, self.lens, self.cu = _dev(tables, dev), _dev(lens, dev), _dev(self.np_cu, dev)
        self.prefix_table = _dev(self.np_prefix, dev)
        self.prefix_len = _dev([prefix], dev)
        self.Q = (q_scale * torch.randn((int(new.sum()), H * G, d), generator=g, device=dev)).to(dtype)

    def run(self, **kw):
        kw.setdefault("return_lse", True)
        Q = kw.pop("Q", self.Q)
        with_prefix = dict(prefix_table=self.prefix_table, prefix_len=self.prefix_len) if self.prefix else {}
        return paged.prefix_attention(Q, self.pool_K, self.pool_V, self.tables, self.lens, self.cu, scale=self.scale,
                                      **with_prefix, **kw)

    def oracle(self):
        return po.prefix_attention(_np(self.Q), _np(self.pool_K), _np(self.pool_V), self.np_tables, self.np_lens,
                                   self.np_cu, self.np_prefix, self.prefix, self.scale)

    def check(self, out, lse, rows=slice(None)):
        o, z, A, top = (x[rows] for x in self.oracle())
        d = self.Q.shape[2]
        n = self.prefix + int(self.np_lens.max())
        u, e = torch.finfo(self.dtype).eps / 2, 2.0 ** -24
        s = (d + 8) * e * top
        per = (0 if self.dtype == F32 else u) + 2 * s[..., None] + 2 * (n * e + 2.0 ** -21)
        got = _np(out)[rows]
        err = np.abs(got - o)
        tol = u * np.abs(o) + per * A
        assert np.isfinite(got).all()
        assert (err <= tol).all(), f"worst {np.max(err / np.maximum(tol, 1e-30)):.3f} of the tolerance"
        if lse is not None:
            got = _np(lse)[rows]
            seen = np.isfinite(z)
            assert np.array_equal(np.isneginf(got), ~seen)
            tol = s + n * e + 2.0 ** -21 + 2 * e * np.abs(np.where(seen, z, 0))
            assert (np.abs(got - z)[seen] <= tol[seen]).all()


SHAPES = [  # lens, new, prefix, H, G, d, L
    ([1], [1], 0, 1, 1, 64, 16),
    ([1], [1], 1, 1, 1, 64, 16),
    ([5, 64, 17], [1, 1, 1], 64, 2, 4, 64, 16),
    ([5, 0, 17], [1, 0, 3], 7, 2, 3, 64, 16),
    ([130, 1, 128, 127, 129], [1, 1, 1, 1, 1], 129, 2, 4, 128, 64),
    ([300, 20, 1], [7, 20, 1], 127, 1, 5, 128, 16),
    ([200, 333], [200, 33], 128, 2, 2, 128, 32),
    ([700], [700], 300, 1, 2, 64, 128),
    ([3, 900, 60, 1, 1, 450], [1, 1, 2, 1, 1, 4], 1000, 2, 8, 128, 64),
    ([40] * 40, [1] * 40, 513, 1, 8, 128, 64),
    ([260, 515], [140, 2], 0, 4, 1, 128, 128),
    ([9, 600], [2, 5], 33, 1, 16, 64, 64),
]


@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
@pytest.mark.parametrize("shape", SHAPES, ids=[f"shape{i}" for i in range(len(SHAPES))])
def test_attention(cuda_device, dtype, shape):
    s = Setup(cuda_device, dtype, *shape, seed=len(shape[0]) + shape[2])
    s.check(*s.run())
    nat.check_device_errors()


@pytest.mark.parametrize("dtype, d, dv, L", [
    (F32, 80, 48, 16), (BF16, 80, 80, 16), (BF16, 256, 256, 64), (FP16, 128, 64, 64), (BF16, 128, 128, 24),
    (BF16, 64, 64, 1), (F32, 4, 4, 5), (FP16, 8, 8, 3), (BF16, 64, 64, 256), (BF16, 128, 128, 8), (F32, 256, 256, 128),
])
def test_attention_other_shapes(cuda_device, dtype, d, dv, L):
    s = Setup(cuda_device, dtype, [70, 1, 200], [3, 1, 60], 150, 2, 3, d, L, dv=dv, seed=d + L)
    s.check(*s.run())


@pytest.mark.parametrize("dtype, d", [(BF16, 128), (FP16, 64), (F32, 128)])
@pytest.mark.parametrize("rows", [3, 16, 17, 32, 33, 64, 100, 128, 129, 256, 257, 300, 385])
def test_rows_of_the_prefix(cuda_device, dtype, d, rows):
    # as many one-token requests as rows: every size of the prefix's last item
    s = Setup(cuda_device, dtype, [1 + i % 70 for i in range(rows)], [1] * rows, 300, 1, 1, d, 32, seed=rows)
    s.check(*s.run())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5])
def test_few_rows_over_long_requests(cuda_device, dtype, G):
    # a block length that the tensor-core kernel does not take, 65 to 128 columns
    s = Setup(cuda_device, dtype, [2000, 33, 1, 400], [1, 1, 1, 1], 0, 2, G, 104, 24, dv=128, seed=G)
    s.check(*s.run())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_output_over_the_queries(cuda_device, dtype):
    s = Setup(cuda_device, dtype, [200, 5], [130, 2], 64, 1, 2, 64, 16, seed=12)
    want, lse = s.run()
    q = s.Q.clone()
    got, lse2 = s.run(Q=q, out=q)
    assert got is q and torch.equal(q, want) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_long_single_request(cuda_device, dtype):
    # one request split over every SM: continuations of the prefix and of the own part
    s = Setup(cuda_device, dtype, [9001], [1], 12345, 1, 4, 128, 64, seed=3)
    s.check(*s.run())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hidden", [float("inf"), float("-inf"), float("nan"), 6e4])
def test_masked_places_may_hold_anything(cuda_device, dtype, hidden):
    s = Setup(cuda_device, dtype, [5, 140, 64], [2, 1, 64], 70, 2, 2, 128, 64, seed=1, hidden=hidden)
    s.check(*s.run())


@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_later_tokens_do_not_reach_earlier_queries(cuda_device, dtype, value):
    # the last new token's key and value are not finite: earlier queries are unaffected
    s = Setup(cuda_device, dtype, [150, 40], [9, 1], 20, 2, 2, 64, 16, seed=4)
    out, lse = s.run()
    p = 149
    blk = int(s.np_tables[0, p // 16])
    s.pool_V[blk, :, p % 16] = value
    s.pool_K[blk, :, p % 16] = value
    again, lse2 = s.run()
    keep = [t for t in range(10) if t != 8]
    assert torch.equal(out[keep], again[keep]) and torch.equal(lse[keep], lse2[keep])
    assert not torch.isfinite(again[8].float()).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_see_nothing(cuda_device, dtype):
    s = Setup(cuda_device, dtype, [4, 20], [2, 3], 0, 2, 2, 64, 16, seed=6)
    s.lens = _dev([1, 20], cuda_device)   # the first new token of request 0 sees nothing
    s.np_lens = np.array([1, 20])
    out, lse = s.run()
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all()
    s.check(out, lse)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_scores(cuda_device, dtype):
    # logits of some hundreds: the running maximum moves late and by much
    s = Setup(cuda_device, dtype, [400, 90], [1, 5], 700, 1, 4, 128, 64, seed=8, q_scale=40.0)
    blk = int(s.np_prefix[9])
    s.pool_K[blk] *= 3
    s.check(*s.run())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_tail_rows(cuda_device, dtype):
    s = Setup(cuda_device, dtype, [30, 7], [2, 1], 40, 2, 2, 64, 16, seed=2)
    Q = torch.cat([s.Q, torch.full((4, 4, 64), float("nan"), dtype=dtype, device=cuda_device)])
    want, want_lse = s.run()
    out, lse = s.run(Q=Q)
    assert torch.equal(out[:3], want) and torch.equal(lse[:3], want_lse)
    assert (out[3:] == 0).all() and torch.isneginf(lse[3:]).all()
    mine = torch.full((7, 4, 64), 5.0, dtype=dtype, device=cuda_device)
    got, _ = s.run(Q=Q, out=mine)
    assert got is mine and torch.equal(mine[:3], want) and (mine[3:] == 5.0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strided_queries_tables_and_default_scale(cuda_device, dtype):
    s = Setup(cuda_device, dtype, [30, 170], [3, 1], 90, 2, 4, 64, 16, seed=11)
    want, want_lse = s.run()
    fused = torch.randn((4, 12, 192), device=cuda_device).to(dtype)
    fused[:, 2:10, 64:128] = s.Q
    wide = torch.full((2, 40), -7, dtype=torch.int32, device=cuda_device)
    wide[:, :s.tables.shape[1]] = s.tables
    s.tables = wide[:, :s.tables.shape[1]]
    out, lse = s.run(Q=fused[:, 2:10, 64:128])
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    s.tables = wide                      # entries behind a request's blocks are not read
    out, lse = s.run(Q=fused[:, 2:10, 64:128])
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    odd = torch.empty(s.Q.numel() + 1, dtype=dtype, device=cuda_device)[1:].view(s.Q.shape).copy_(s.Q)
    out, _ = s.run(Q=odd)                # 2- or 4-byte aligned
    assert torch.equal(out, want)
    s.scale = None
    out, lse = s.run()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    out, lse = s.run(return_lse=False)
    assert torch.equal(out, want) and lse is None


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bad_table_entries_are_reported(cuda_device, dtype):
    s = Setup(cuda_device, dtype, [50, 70], [1, 1], 40, 1, 2, 64, 16, seed=12)
    want, _ = s.run()
    s.tables[0, 1] = 10 ** 9
    out, _ = s.run()
    with pytest.raises(RuntimeError, match="table entry"):
        nat.check_device_errors()
    assert torch.equal(out[1], want[1])
    s.tables[0, 1] = -1
    s.run()
    with pytest.raises(RuntimeError, match="table entry"):
        nat.check_device_errors()
    nat.check_device_errors()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_lengths_beyond_the_tables_are_cut(cuda_device, dtype):
    s = Setup(cuda_device, dtype, [48, 32], [1, 1], 32, 1, 2, 64, 16, seed=13)
    want, lse = s.run()
    s.lens, s.prefix_len = _dev([10 ** 9, 32], cuda_device), _dev([2 ** 31 - 1], cuda_device)
    out, lse2 = s.run()
    assert torch.equal(out, want) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_odd_offsets_stay_in_bounds(cuda_device, dtype):
    # offsets that do not ascend, or leave the packed rows: no fault, and rows of sound requests are right
    s = Setup(cuda_device, dtype, [20, 33, 5], [2, 1, 1], 40, 1, 2, 64, 16, seed=14)
    for cu in ([0, 2, 1, 4], [0, -5, 9, 2 ** 31 - 1], [3, 2, 1, 0], [2 ** 31 - 1] * 4, [-1, -1, -1, -1]):
        s.cu = _dev(cu, cuda_device)
        out, lse = s.run()
        assert out.shape == (4, 2, 64)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_more_than_2_31_elements(cuda_device, dtype):
    # blocks beyond 2^31 elements of the pool
    H, L, d = 8, 64, 128
    F = 36000 if dtype == F32 else 70000
    pool_K = torch.empty((F, H, L, d), dtype=dtype, device=cuda_device)
    pool_V = torch.empty_like(pool_K)
    small = Setup(cuda_device, dtype, [100, 64], [1, 2], 150, H, 2, d, L, seed=15)
    want, want_lse = small.run()
    n = small.pool_K.shape[0]
    pool_K[F - n:], pool_V[F - n:] = small.pool_K, small.pool_V
    out, lse = paged.prefix_attention(
        small.Q, pool_K, pool_V, torch.where(small.tables >= 0, small.tables + (F - n), small.tables), small.lens,
        small.cu, prefix_table=small.prefix_table + (F - n), prefix_len=small.prefix_len, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    rows = torch.randn((2, H, d), device=cuda_device).to(dtype)
    slots = _dev([F * L - 1, (F - 1) * L], cuda_device)
    paged.paged_append(rows, rows, pool_K, pool_V, slots)
    assert torch.equal(pool_K[F - 1, :, L - 1], rows[0]) and torch.equal(pool_V[F - 1, :, 0], rows[1])


def test_attention_is_repeatable(cuda_device):
    for dtype in (BF16, F32):
        s = Setup(cuda_device, dtype, [3, 900, 60, 450], [1, 1, 2, 4], 5000, 2, 8, 128, 64, seed=16)
        out, lse = s.run()
        for _ in range(3):
            again, lse2 = s.run()
            assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_two_streams_at_once(cuda_device):
    a = Setup(cuda_device, BF16, [300, 900], [1, 2], 2000, 2, 4, 128, 64, seed=17)
    b = Setup(cuda_device, BF16, [77, 1, 600], [3, 1, 1], 700, 2, 4, 128, 64, seed=18)
    want = [a.run(), b.run()]
    s1, s2 = torch.cuda.Stream(cuda_device), torch.cuda.Stream(cuda_device)
    got = []
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s1):
            x = a.run()
        with torch.cuda.stream(s2):
            y = b.run()
        got.append((x, y))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x[0], want[0][0]) and torch.equal(y[0], want[1][0])


def test_attention_refuses(cuda_device):
    s = Setup(cuda_device, BF16, [30, 7], [2, 1], 40, 2, 2, 64, 16, seed=2)
    call = lambda **kw: paged.prefix_attention(  # noqa: E731
        **{**dict(Q=s.Q, pool_K=s.pool_K, pool_V=s.pool_V, tables=s.tables, lens=s.lens, cu_new=s.cu), **kw})
    with pytest.raises(RuntimeError, match="mixed"):
        call(Q=s.Q.float())
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        call(Q=s.Q.double(), pool_K=s.pool_K.double(), pool_V=s.pool_V.double())
    with pytest.raises(ValueError):
        call(Q=s.Q[:, :3])
    with pytest.raises(ValueError):
        call(Q=s.Q[:, :, :32])
    with pytest.raises(ValueError):
        call(lens=s.lens[:1])
    with pytest.raises(ValueError):
        call(cu_new=s.cu[:2])
    with pytest.raises(RuntimeError, match="int32"):
        call(tables=s.tables.long())
    with pytest.raises(ValueError, match="together"):
        call(prefix_table=s.prefix_table)
    with pytest.raises(ValueError, match="out"):
        call(out=torch.empty((3, 4, 32), dtype=BF16, device=cuda_device))
    with pytest.raises(ValueError, match="finite"):
        call(scale=float("nan"))
    with pytest.raises(RuntimeError, match="backward"):
        call(Q=s.Q.clone().requires_grad_())
    with pytest.raises(ValueError, match="contiguous"):
        call(pool_K=s.pool_K.transpose(1, 2).contiguous().transpose(1, 2))
    big = torch.zeros((2, 1, 16, 264), dtype=BF16, device=cuda_device)
    with pytest.raises(RuntimeError, match="unsupported shape"):
        call(Q=torch.zeros((3, 1, 264), dtype=BF16, device=cuda_device), pool_K=big, pool_V=big)


def test_empty_calls(cuda_device):
    s = Setup(cuda_device, BF16, [30, 7], [0, 0], 40, 2, 2, 64, 16, seed=2)
    out, lse = s.run()
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    out, lse = s.run(Q=torch.ones((3, 4, 64), dtype=BF16, device=cuda_device))
    assert (out == 0).all() and torch.isneginf(lse).all()


# ---------------------------------------------------------------------------
# together: a serving loop
# ---------------------------------------------------------------------------
class Recount:
    """The same loop with Python lists of key and value rows per request."""

    def __init__(self, n):
        self.K, self.V = [[] for _ in range(n)], [[] for _ in range(n)]
        self.pK, self.pV = [], []

    def step(self, new, K, V, Q, G, scale):
        at, outs = 0, []
        for b, n in enumerate(new):
            if n < 0:
                self.K[b], self.V[b] = [], []
            for _ in range(max(n, 0)):
                self.K[b].append(K[at])
                self.V[b].append(V[at])
                k, v = np.stack(self.pK + self.K[b]), np.stack(self.pV + self.V[b])   # [n, H, d]
                o = []
                for hq in range(Q.shape[1]):
                    s = k[:, hq // G] @ Q[at, hq] * scale
                    p = np.exp(s - s.max())
                    o.append(p @ v[:, hq // G] / p.sum())
                outs.append(np.stack(o))
                at += 1
        return np.stack(outs) if outs else np.zeros((0, *Q.shape[1:]))


@pytest.mark.parametrize("dtype, d, L", [(BF16, 64, 16), (FP16, 128, 32), (F32, 64, 16)])
def test_serving_loop(cuda_device, dtype, d, L):
    H, G, R = 2, 2, 5
    rng = np.random.default_rng(d)
    g = torch.Generator(device=cuda_device).manual_seed(d)
    mem = paged.PagedMemory(60, L, H, d, max_requests=R, max_blocks=12, n_layers=2, dtype=dtype, device=cuda_device)
    ref = Recount(R)

    def step(new, pad=0):
        n = int(np.maximum(new, 0).sum())
        make = lambda h: torch.randn((n + pad, h, d), generator=g, device=cuda_device).to(dtype)  # noqa: E731
        K, V, Q = make(H), make(H), make(H * G)
        t = mem.extend(_dev(new, cuda_device), n + pad)
        mem.append(V, K, t, layer=0)
        mem.append(K, V, t, layer=1)
        out, _ = mem.attend(Q, t, layer=1)
        assert int(t.n_short) == 0 and int(t.cu_new[-1]) == n
        want = ref.step(new, _np(K), _np(V), _np(Q), G, d ** -0.5)
        # half a step of the output and of the weights, |o| and A below 4 here; fp32: sums of 300 terms
        tol = 8 * torch.finfo(dtype).eps / 2 if dtype != F32 else 300 * 8 * 2.0 ** -24
        assert np.abs(_np(out)[:n] - want).max(initial=0) <= tol
        assert (_np(out)[n:] == 0).all()

    step(np.array([3 * L + 5, 0, 0, 0, 0]))
    mem.share(0)
    ref.pK, ref.pV, ref.K[0], ref.V[0] = ref.K[0], ref.V[0], [], []
    step(np.array([0, L + 1, 2, 1, 0]), pad=3)
    for i in range(6):
        step(np.array([1, 1, 1, 1, 1 if i else 4]), pad=i)
    step(np.array([1, -1, 1, -1, 5]))
    for i in range(5):
        step(rng.integers(0, 4, R))
    step(np.array([-1, 2 * L, -1, 1, -1]))
    held = int((mem.tables >= 0).sum()) + int((mem.prefix_table >= 0).sum())
    assert held + int(mem.free_state[1]) == 60
    mem.unshare(0)
    ref.K[0], ref.V[0], ref.pK, ref.pV = ref.pK, ref.pV, [], []
    step(np.array([1, 1, 0, 0, 2]))
    step(np.array([-1] * 5))
    assert int(mem.free_state[1]) == 60 and int((mem.tables >= 0).sum()) == 0
    with pytest.raises(ValueError):
        mem.share(R)
    mem.reset()
    assert mem.free_ring.tolist() == list(range(60))


def test_share_refuses_a_second_prefix(cuda_device):
    mem = paged.PagedMemory(8, 16, 1, 64, max_requests=2, max_blocks=4, device=cuda_device)
    mem.extend(_dev([3, 2], cuda_device), 5)
    mem.share(0)
    with pytest.raises(RuntimeError, match="prefix already"):
        mem.share(1)
    with pytest.raises(RuntimeError, match="holds tokens"):
        mem.unshare(1)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_captured_step_replays_with_other_lengths(cuda_device, dtype):
    H, G, d, L, R, N = 2, 4, 64, 16, 6, 16
    g = torch.Generator(device=cuda_device).manual_seed(1)
    make = lambda h: torch.randn((N, h, d), generator=g, device=cuda_device).to(dtype)  # noqa: E731

    def fresh():
        m = paged.PagedMemory(40, L, H, d, max_requests=R, max_blocks=5, dtype=dtype, device=cuda_device)
        t = m.extend(_dev([20, 0, 0, 0, 0, 0], cuda_device), 20)
        gg = torch.Generator(device=cuda_device).manual_seed(2)
        kv = torch.randn((20, H, d), generator=gg, device=cuda_device).to(dtype)
        m.append(kv, kv, t)
        m.share(0)
        return m

    eager, captured = fresh(), fresh()
    new, K, V, Q = _dev([1] * R, cuda_device), make(H), make(H), make(H * G)

    def one(m, new, K, V, Q):
        t = m.extend(new, N)
        m.append(K, V, t)
        return m.attend(Q, t, return_lse=True)

    warm = fresh()
    side = torch.cuda.Stream(cuda_device)
    with torch.cuda.stream(side):
        one(warm, new, K, V, Q)
    torch.cuda.synchronize()
    # two graphs on one memory, replayed in turn
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = one(captured, new, K, V, Q)
        graphs.append((gr, res))
    for i, lens in enumerate([[1] * R, [3, 0, 1, 2, 0, 1], [0, 9, 0, 0, 5, 0], [-1, 1, 1, -1, 1, 1], [2, 2, 2, 2, 2, 2]]):
        new.copy_(_dev(lens, cuda_device))
        K.copy_(make(H)), V.copy_(make(H)), Q.copy_(make(H * G))
        gr, res = graphs[i % 2]
        gr.replay()
        want = one(eager, new, K, V, Q)
        assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])
        assert torch.equal(captured.tables, eager.tables) and torch.equal(captured.lens, eager.lens)
        assert torch.equal(captured.free_ring, eager.free_ring)
