"""Paged block memory without a GPU: the refusals of the C entry points and of
the Python operators, and the oracle of the block tables against a recount."""
import ctypes

import numpy as np
import pytest
import torch

from gfst_hmb_public_b200 import _native as nat
from gfst_hmb_public_b200 import paged
from oracle import paged_oracle as po

FAKE = 4096  # a 16-byte aligned address that no refused call dereferences


def _tables(**kw):
    a = dict(lens=FAKE, new=FAKE * 2, tables=FAKE * 3, ring=FAKE * 4, state=FAKE * 5, B=4, W=8, L=16, F=64, n=10,
             t_out=FAKE * 6, l_out=FAKE * 7, cu=FAKE * 8, slots=FAKE * 9, s_out=FAKE * 10, short=FAKE * 11)
    a.update(kw)
    return nat.load().gfst_block_tables(a["lens"], a["new"], a["tables"], a["ring"], a["state"], a["B"], a["W"],
                                        a["L"], a["F"], a["n"], a["t_out"], a["l_out"], a["cu"], a["slots"],
                                        a["s_out"], a["short"], None)


@pytest.mark.parametrize("kw, status", [
    (dict(B=0), 2), (dict(B=16385), 2), (dict(W=0), 2), (dict(L=0), 2), (dict(W=1 << 20, L=1 << 12), 2),
    (dict(F=0), 2), (dict(F=1 << 28), 2), (dict(n=-1), 2), (dict(n=1 << 31), 2), (dict(lens=None), 1),
    (dict(new=None), 1), (dict(tables=None), 1), (dict(ring=None), 1), (dict(state=None), 1), (dict(t_out=None), 1),
    (dict(l_out=None), 1), (dict(cu=None), 1), (dict(slots=None), 1), (dict(s_out=None), 1), (dict(short=None), 1),
    (dict(l_out=FAKE), 1), (dict(l_out=FAKE * 2), 1), (dict(s_out=FAKE * 5), 1),
])
def test_block_tables_refuses(kw, status):
    assert _tables(**kw) == status
    assert nat.load().gfst_last_error()


def _append(**kw):
    a = dict(K=FAKE, kt=256, kh=128, V=FAKE, vt=256, vh=128, pk=FAKE, pv=FAKE, slots=FAKE, n=4, F=8, L=16, H=2, d=128,
             dv=128, dt=nat.DTYPE_BF16)
    a.update(kw)
    return nat.load().gfst_paged_append(a["K"], a["kt"], a["kh"], a["V"], a["vt"], a["vh"], a["pk"], a["pv"],
                                        a["slots"], a["n"], a["F"], a["L"], a["H"], a["d"], a["dv"], a["dt"], None)


@pytest.mark.parametrize("kw, status", [
    (dict(dt=nat.DTYPE_F64), 7), (dict(dt=9), 7), (dict(n=-1), 2), (dict(F=0), 2), (dict(L=0), 2), (dict(H=0), 2),
    (dict(d=0), 2), (dict(F=1 << 28), 2), (dict(d=12), 3), (dict(dv=4), 3), (dict(K=None), 1), (dict(V=None), 1),
    (dict(pk=None), 1), (dict(pv=None), 1), (dict(slots=None), 1), (dict(K=FAKE + 8), 3), (dict(pv=FAKE + 2), 3),
    (dict(kt=260), 3), (dict(vh=4), 3),
])
def test_paged_append_refuses(kw, status):
    assert _append(**kw) == status


def test_paged_append_of_nothing():
    assert _append(n=0, K=None, V=None, slots=None) == 0


def _attend(**kw):
    a = dict(Q=FAKE, qt=1024, qh=128, pk=FAKE, pv=FAKE, F=8, L=16, H=2, G=4, d=128, dv=128, dt=nat.DTYPE_BF16,
             tables=FAKE, ts=8, W=8, lens=FAKE, cu=FAKE, B=2, n=2, pt=FAKE, P=2, pl=FAKE, scale=0.1, out=FAKE,
             lse=None, fill=1, ws=FAKE, wb=1 << 40)
    a.update(kw)
    return nat.load().gfst_prefix_attention(
        a["Q"], a["qt"], a["qh"], a["pk"], a["pv"], a["F"], a["L"], a["H"], a["G"], a["d"], a["dv"], a["dt"],
        a["tables"], a["ts"], a["W"], a["lens"], a["cu"], a["B"], a["n"], a["pt"], a["P"], a["pl"], a["scale"],
        a["out"], a["lse"], a["fill"], a["ws"], a["wb"], None)


@pytest.mark.parametrize("kw, status", [
    (dict(dt=nat.DTYPE_F64), 7), (dict(H=0), 2), (dict(G=0), 2), (dict(d=0), 2), (dict(d=264), 2), (dict(dv=264), 2),
    (dict(d=12), 3), (dict(dv=4), 3), (dict(B=0), 2), (dict(B=65537), 2), (dict(W=0), 2), (dict(L=0), 2),
    (dict(F=0), 2), (dict(P=-1), 2), (dict(n=-1), 2), (dict(n=1 << 30), 2), (dict(W=1 << 30), 2), (dict(P=1 << 30), 2),
    (dict(Q=None), 1), (dict(pk=None), 1), (dict(pv=None), 1), (dict(tables=None), 1), (dict(lens=None), 1),
    (dict(cu=None), 1), (dict(out=None), 1), (dict(ws=None), 1), (dict(pt=None), 1), (dict(pl=None), 1),
    (dict(Q=FAKE + 4), 3), (dict(qt=1028), 3), (dict(qh=4), 3), (dict(out=FAKE + 8), 3), (dict(ws=FAKE + 16), 3),
    (dict(wb=1000), 2),
])
def test_prefix_attention_refuses(kw, status):
    assert _attend(**kw) == status


@pytest.mark.parametrize("kw, status", [
    # the last position of a tile of 128 keys passes 2^31
    (dict(W=(1 << 31) - 512, L=1), 2), (dict(P=(1 << 31) - 512, L=1), 2), (dict(W=(1 << 27) - 1), 2),
    (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1), (dict(scale=3e38), 1), (dict(scale=-3e38), 1),
])
def test_prefix_attention_refuses_far_positions_and_scales(kw, status):
    assert _attend(**kw) == status


def test_prefix_attention_of_nothing():
    assert _attend(n=0, Q=None, out=None, ws=None) == 0


def test_workspace_grows_with_the_rows():
    lib, n = nat.load(), ctypes.c_size_t(0)
    sizes = []
    for tokens in (1, 64, 4096):
        assert lib.gfst_prefix_attention_workspace_bytes(tokens, 8, 4, 128, ctypes.byref(n)) == 0
        sizes.append(n.value)
    assert sizes[0] < sizes[1] < sizes[2] and all(s % 256 == 0 for s in sizes)
    assert lib.gfst_prefix_attention_workspace_bytes(-1, 8, 4, 128, ctypes.byref(n)) == 2
    assert lib.gfst_prefix_attention_workspace_bytes(4, 8, 4, 128, None) == 1


def test_operators_refuse_cpu_tensors():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    x = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    pool = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.block_tables(i(2), i(2), i(2, 4), i(8), i(2), block_len=16, n_tokens=2)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.paged_append(x, x, pool, pool, i(2))
    with pytest.raises(RuntimeError, match="CUDA"):
        paged.prefix_attention(x, pool, pool, i(2, 4), i(2), i(3))


def test_memory_refuses_sizes_and_types():
    with pytest.raises(ValueError):
        paged.PagedMemory(0, 16, 2, 64, max_requests=2, max_blocks=4, device="cpu")
    with pytest.raises(RuntimeError):
        paged.PagedMemory(4, 16, 2, 64, max_requests=2, max_blocks=4, dtype=torch.float64, device="cpu")


@pytest.mark.parametrize("seed", range(6))
def test_oracle_tables_conserve_blocks(seed):
    rng = np.random.default_rng(seed)
    B, W, L, F = 5, 6, int(rng.integers(1, 9)), 40
    tables, lens = np.full((B, W), -1), np.zeros(B, dtype=np.int64)
    ring, state = rng.permutation(F), np.array([int(rng.integers(F)), F])
    for _ in range(12):
        new = np.minimum(rng.integers(-1, 2 * L, B), W * L - lens)
        tables, lens, cu, slots, state, short, ring = po.block_tables(lens, new, tables, ring, state, L, 100)
        held = tables[tables >= 0].tolist()
        free = [int(ring[(state[0] + i) % F]) for i in range(state[1])]
        assert short == 0 and sorted(held + free) == list(range(F))
        assert len(set(slots[slots >= 0].tolist())) == cu[-1]


@pytest.mark.parametrize("seed", range(4))
def test_oracle_attention_against_a_dense_softmax(seed):
    rng = np.random.default_rng(seed)
    H, G, d, L, P = 2, 3, 8, 4, int(rng.integers(0, 11))
    pool_K, pool_V = rng.standard_normal((2, 12, H, L, d))
    tables, lens, cu = np.array([[5, 1, 7], [9, -1, -1]]), np.array([10, 3]), np.array([0, 4, 5])
    Q = rng.standard_normal((6, H * G, d))
    out, lse, mean_abs, top = po.prefix_attention(Q, pool_K, pool_V, tables, lens, cu, np.array([0, 2, 3]), P, 0.3)
    for t, (b, see) in enumerate([(0, 7), (0, 8), (0, 9), (0, 10), (1, 3)]):
        for h in range(H * G):
            rows = [pool_K[[0, 2, 3][p // L], h // G, p % L] for p in range(P)]
            rows += [pool_K[tables[b, p // L], h // G, p % L] for p in range(see)]
            vals = [pool_V[[0, 2, 3][p // L], h // G, p % L] for p in range(P)]
            vals += [pool_V[tables[b, p // L], h // G, p % L] for p in range(see)]
            s = np.stack(rows) @ Q[t, h] * 0.3
            w = np.exp(s - s.max())
            assert np.allclose(out[t, h], w @ np.stack(vals) / w.sum(), rtol=1e-12, atol=1e-12)
            assert np.isclose(lse[t, h], s.max() + np.log(w.sum()))
            assert np.allclose(mean_abs[t, h], w @ np.abs(np.stack(vals)) / w.sum())
    assert (out[5] == 0).all() and np.isneginf(lse[5]).all()


@pytest.mark.parametrize("status", [0, 2, 7, 8, -1])
def test_debug_attention_error_refuses_other_statuses(status):
    assert nat.load().gfst_debug_attention_error(1, status, None) == 1


def test_gradients_of_either_mode_are_refused():
    # the operators' own check, which asks no device
    x, y = torch.ones(3), torch.ones(3, requires_grad=True)
    paged._no_grad("op", x, None)
    with pytest.raises(RuntimeError, match="backward"):
        paged._no_grad("op", x, y)
    with torch.no_grad():
        paged._no_grad("op", x, y)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        paged._no_grad("op", x)
        with pytest.raises(RuntimeError, match="forward-mode"):
            paged._no_grad("op", x, dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            paged._no_grad("op", dual)
        with torch.inference_mode():
            paged._no_grad("op", dual)


def test_pools_without_heads_are_refused():
    pool, x = torch.zeros((4, 0, 16, 64)), torch.zeros((2, 2, 64))
    with pytest.raises(ValueError, match="heads"):
        paged._check_pools("prefix_attention", pool, pool)
