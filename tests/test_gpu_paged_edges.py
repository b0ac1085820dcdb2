"""Paged block memory on the GPU: calls at the edges of what its documentation
allows.  Tolerances as in test_gpu_paged.py (``Setup.check``)."""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from gfst_hmb_public_b200 import _native as nat
from gfst_hmb_public_b200 import paged
from test_gpu_paged import BF16, F32, FP16, Setup, _dev

pytestmark = pytest.mark.gpu

REPO = Path(__file__).resolve().parents[1]


def _soil(dev, floats):
    """Leave numbers where the next allocation of that size begins."""
    held = [torch.full((floats,), 7.0, device=dev) for _ in range(4)]
    del held


@pytest.mark.parametrize("dtype, d, G", [(BF16, 128, 1), (FP16, 64, 1), (BF16, 64, 2), (FP16, 128, 2)])
def test_many_one_tile_parts_of_few_rows_in_a_row(cuda_device, dtype, d, G):
    # a worker takes some dozen parts of one or two rows and one tile each, one
    # right behind the other: no row takes its neighbour's references and sums
    rng = np.random.default_rng(G)
    lens = rng.integers(1, 129, 1500)
    s = Setup(cuda_device, dtype, lens, [1] * 1500, 0, 2, G, d, 64, seed=d + G)
    out, lse = s.run()
    s.check(out, lse)
    for _ in range(5):
        again, lse2 = s.run()
        assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_log_sum_exp_of_padding_beside_a_given_out(cuda_device, dtype):
    # ``out`` keeps its padding rows, the log-sum-exp is -inf there all the same
    s = Setup(cuda_device, dtype, [30, 7], [2, 1], 40, 2, 2, 64, 16, seed=2)
    Q = torch.cat([s.Q, torch.full((4, 4, 64), float("nan"), dtype=dtype, device=cuda_device)])
    want, want_lse = s.run()
    mine = torch.full((7, 4, 64), 5.0, dtype=dtype, device=cuda_device)
    _soil(cuda_device, 7 * 4)
    got, lse = s.run(Q=Q, out=mine)
    assert got is mine and torch.equal(mine[:3], want) and (mine[3:] == 5.0).all()
    assert torch.equal(lse[:3], want_lse) and torch.isneginf(lse[3:]).all()


def test_log_sum_exp_of_a_short_step_beside_a_given_out(cuda_device):
    mem = paged.PagedMemory(2, 16, 1, 64, max_requests=2, max_blocks=4, device=cuda_device)
    t = mem.extend(_dev([40, 1], cuda_device), 41)
    mine = torch.full((41, 2, 64), 5.0, dtype=BF16, device=cuda_device)
    _soil(cuda_device, 41 * 2)
    _, lse = mem.attend(torch.ones((41, 2, 64), dtype=BF16, device=cuda_device), t, out=mine, return_lse=True)
    assert int(t.n_short) == 2 and (mine == 5.0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("B", [4029, 4030, 4095, 4096])
def test_block_tables_around_48_kb_of_sums(cuda_device, B):
    # in a process of its own: a larger call would have asked for the shared memory
    code = (f"import sys; sys.path[:0] = {[str(REPO), str(REPO / 'tests')]!r}\n"
            "import numpy as np, torch\n"
            "from test_gpu_paged import _check_tables, _table_inputs\n"
            f"inputs = _table_inputs(np.random.default_rng({B}), {B}, 5, 16, 60, 9, 0.1, 3)\n"
            "for in_place in (False, True):\n"
            "    _check_tables(torch.device('cuda:0'), inputs, 16, int(np.maximum(inputs[1], 0).sum()), in_place)\n")
    run = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [1, 5, 20, 47])
def test_fewer_packed_rows_than_new_tokens(cuda_device, dtype, rows):
    # the offsets count tokens whose queries are not there: the others see what they would see beside them
    s = Setup(cuda_device, dtype, [90, 200], [8, 40], 33, 2, 4, 64, 16, seed=21)
    out, lse = s.run(Q=s.Q[:rows])
    assert out.shape[0] == rows
    s.check(out, lse, slice(0, rows))


def test_step_in_place_with_fewer_rows_than_tokens_changes_nothing(cuda_device):
    mem = paged.PagedMemory(12, 16, 1, 64, max_requests=3, max_blocks=5, device=cuda_device)
    x = torch.randn((40, 1, 64), device=cuda_device).to(BF16)
    mem.append(x, x, mem.extend(_dev([30, 10, 0], cuda_device), 40))
    kept = (mem.tables, mem.lens, mem.free_ring, mem.free_state, mem.pool_K)
    before = [t.clone() for t in kept]
    new = _dev([3, -1, 18], cuda_device)
    for n in (20, 3, 0):                                        # 21 tokens
        t = mem.extend(new, n)
        mem.append(x[:n], x[:n], t)
        out, lse = mem.attend(torch.ones((n, 2, 64), dtype=BF16, device=cuda_device), t, return_lse=True)
        assert int(t.n_short) == 21 - n
        assert (t.cu_new == 0).all() and (t.slot_map == -1).all()
        assert all(torch.equal(a, b) for a, b in zip(before, kept))
        assert (out == 0).all() and torch.isneginf(lse).all()
    t = mem.extend(new, 21)
    assert int(t.n_short) == 0 and mem.lens.tolist() == [33, 0, 18]


ARG, ALIGN, TIMEOUT = 1, 3, 6


@pytest.mark.parametrize("recorded, reported", [
    ([(1, TIMEOUT), (1, ARG)], TIMEOUT), ([(1, ARG), (1, TIMEOUT)], TIMEOUT), ([(0, ARG), (1, TIMEOUT)], TIMEOUT),
    ([(0, ARG), (1, ARG)], ARG), ([(0, ARG)], ARG), ([(1, ARG)], ARG), ([(1, ALIGN), (1, ARG), (0, ARG)], ALIGN),
    ([(1, TIMEOUT), (0, ARG), (1, ALIGN)], TIMEOUT),
])
def test_a_bad_table_entry_hides_nothing(cuda_device, recorded, reported):
    lib, stream = nat.load(), torch.cuda.current_stream(cuda_device).cuda_stream
    nat.check_device_errors()
    for tensor_cores, status in recorded:
        assert lib.gfst_debug_attention_error(tensor_cores, status, stream) == 0
    assert lib.gfst_check_device_errors(0) == reported
    text = {ARG: "table entry", ALIGN: "shared memory misaligned", TIMEOUT: "bounded wait"}[reported]
    with pytest.raises(RuntimeError, match=text):
        nat.check_device_errors()
    nat.check_device_errors()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_bad_table_entry_behind_a_wait_that_gave_up(cuda_device, dtype):
    # the same by the kernels themselves: a launch that meets a bad entry after the status of another one
    s = Setup(cuda_device, dtype, [50], [1], 0, 1, 2, 64, 16, seed=12)
    s.tables[0, 1] = -1
    stream = torch.cuda.current_stream(cuda_device).cuda_stream
    assert nat.load().gfst_debug_attention_error(int(dtype == BF16), TIMEOUT, stream) == 0
    s.run()
    with pytest.raises(RuntimeError, match="bounded wait"):
        nat.check_device_errors()
    nat.check_device_errors()


def test_tangents_and_a_differentiable_out_are_refused(cuda_device):
    s = Setup(cuda_device, BF16, [30, 7], [2, 1], 40, 2, 2, 64, 16, seed=2)
    out = torch.zeros((3, 4, 64), dtype=BF16, device=cuda_device)
    with pytest.raises(RuntimeError, match="backward"):
        s.run(out=out.clone().requires_grad_())
    K = torch.ones((2, 2, 64), dtype=BF16, device=cuda_device)
    slots, before = _dev([0, 1], cuda_device), s.pool_K.clone()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual
        with pytest.raises(RuntimeError, match="forward-mode"):
            s.run(Q=dual(s.Q, s.Q))
        with pytest.raises(RuntimeError, match="forward-mode"):
            s.run(out=dual(out, out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            paged.paged_append(dual(K, K), K, s.pool_K, s.pool_V, slots)
    assert torch.equal(s.pool_K.nan_to_num(), before.nan_to_num())
    with pytest.raises(RuntimeError):                           # transforms hand over no memory
        torch.func.jvp(lambda q: s.run(Q=q)[0], (s.Q,), (s.Q,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda q: s.run(Q=q)[0])(torch.stack([s.Q, s.Q]))


# ---------------------------------------------------------------------------
# long lengths: a table that lists a few blocks again and again
# ---------------------------------------------------------------------------
class Repeated:
    """Keys and values of ``cycle`` positions, which a long table repeats.  The
    oracle weighs each of them by how often a row sees it."""

    def __init__(self, dev, dtype, H, G, n, d, L, blocks, dv=None, positive=False, seed=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        dv = d if dv is None else dv
        self.pool_K = torch.randn((blocks, H, L, d), generator=g, device=dev).to(dtype)
        self.pool_V = torch.randn((blocks, H, L, dv), generator=g, device=dev)
        self.pool_V = (self.pool_V.abs() if positive else self.pool_V).to(dtype)
        self.Q = torch.randn((n, H * G, d), generator=g, device=dev).to(dtype)
        self.dev, self.dtype, self.G, self.L, self.blocks, self.scale = dev, dtype, G, L, blocks, d ** -0.5

    def table(self, length):
        t = torch.arange(-(-length // self.L), dtype=torch.int32, device=self.dev) % self.blocks
        return t.to(torch.int32)

    def run(self, prefix, own):
        """All queries are the last tokens of one request of ``own`` positions."""
        n, i32 = self.Q.shape[0], dict(dtype=torch.int32, device=self.dev)
        tables = self.table(max(own, 1))[None]
        return paged.prefix_attention(self.Q, self.pool_K, self.pool_V, tables, torch.tensor([own], **i32),
                                      torch.tensor([0, n], **i32), prefix_table=self.table(max(prefix, 1)),
                                      prefix_len=torch.tensor([prefix], **i32), return_lse=True)

    def check(self, out, lse, prefix, own, heads):
        """Tolerances as in test_gpu_paged.py, with pieces of at most m = 65,536
        keys, j of them: numerator's sums m 2^-23 (the tensor cores cut off where
        FP32 rounds), denominator's m 2^-24, and j 2^-24 for their joining."""
        n, G, L = self.Q.shape[0], self.G, self.L
        cycle, u = self.blocks * L, torch.finfo(self.dtype).eps / 2
        at = np.arange(cycle)
        times = lambda length: np.maximum(0, (length - 1 - at) // cycle + 1)  # noqa: E731
        for h in heads:
            k = self.pool_K[:, h].double().cpu().numpy().reshape(cycle, -1)
            v = self.pool_V[:, h].double().cpu().numpy().reshape(cycle, -1)
            for t in range(n):
                count = times(prefix) + times(max(0, own - n + t + 1))
                q = self.Q[t, h * G:(h + 1) * G].double().cpu().numpy()
                s = q @ k.T * self.scale
                m = s.max(1, keepdims=True)
                p = np.exp(s - m) * count
                l = p.sum(1, keepdims=True)
                want, A, z = p @ v / l, p @ np.abs(v) / l, m[:, 0] + np.log(l[:, 0])
                top = self.scale * (np.abs(q) @ np.abs(k).T).max(1)
                e, most = 2.0 ** -24, min(65536, max(prefix, own))
                sums = 3 * most * e + (prefix + own) / 65536 * e
                err_s = (q.shape[1] + 8) * e * top
                per = (0 if self.dtype == F32 else u) + 2 * err_s + sums + 2.0 ** -20
                got = out[t, h * G:(h + 1) * G].double().cpu().numpy()
                assert (np.abs(got - want) <= u * np.abs(want) + per[:, None] * A).all()
                got = lse[t, h * G:(h + 1) * G].double().cpu().numpy()
                assert (np.abs(got - z) <= err_s + sums + 2.0 ** -20 + 2 * e * np.abs(z)).all()


@pytest.mark.parametrize("dtype, G, n, d, dv", [
    (BF16, 1, 1, 64, 64), (FP16, 8, 3, 128, 128), (BF16, 8, 5, 64, 64), (BF16, 8, 32, 64, 64),     # tensor cores
    (F32, 1, 1, 64, 64), (F32, 3, 1, 64, 64), (F32, 6, 1, 64, 64), (F32, 8, 3, 64, 64), (F32, 16, 4, 64, 64),
    (BF16, 2, 1, 80, 48), (F32, 2, 1, 136, 136),                                                    # FP32 units
])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_parts_in_pieces(cuda_device, dtype, G, n, d, dv, where):
    # as many heads as workers: a part is a whole item, of three pieces and a bit
    s = Repeated(cuda_device, dtype, 300, G, n, d, 128, 4, dv=dv, seed=G + n)
    prefix, own = (200_001, 40) if where == "prefix" else (0, 200_001)
    out, lse = s.run(prefix, own)
    s.check(out, lse, prefix, own, (0, 150, 299))
    again, lse2 = s.run(prefix, own)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_long_sums_of_one_sign(cuda_device, dtype):
    # in one go, the tensor cores' sums of 8 M positive terms come out 4 % too small
    s = Repeated(cuda_device, dtype, 300, 1, 1, 64, 128, 8, positive=True, seed=3)
    out, lse = s.run(1 << 23, 0)
    s.check(out, lse, 1 << 23, 0, (0, 299))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_positions_up_to_the_last(cuda_device, dtype, where):
    # the most positions that a table can hold: 2^31 - 1024
    s = Repeated(cuda_device, dtype, 1, 4, 1, 64, 1024, 2, seed=4)
    most = (1 << 31) - 1024
    prefix, own = (most, 1) if where == "prefix" else (0, most)
    out, lse = s.run(prefix, own)
    s.check(out, lse, prefix, own, (0,))
    nat.check_device_errors()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_odd_offsets_leave_sound_rows_right(cuda_device, dtype):
    s = Setup(cuda_device, dtype, [20, 33, 5], [2, 1, 1], 40, 1, 2, 64, 16, seed=14)
    tables, lens = s.np_tables, s.np_lens
    # token 0 is request 0's first, tokens 2 and 3 are request 2's last of three; both claim token 1
    s.cu = _dev([0, 2, 1, 4], cuda_device)
    out, lse = s.run()
    for b, cu, rows in ((0, [0, 2], [0]), (2, [1, 4], [2, 3])):
        s.np_tables, s.np_lens, s.np_cu = tables[b:b + 1], lens[b:b + 1], np.array(cu)
        s.check(out, lse, rows)
    # no token is anyone's
    for cu in ([3, 2, 1, 0], [2 ** 31 - 1] * 4, [-1, -1, -1, -1]):
        s.cu = _dev(cu, cuda_device)
        out, lse = s.run()
        assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_most_requests_on_one_table_row(cuda_device, dtype):
    # 65,536 requests, every third idle, all of whose rows of the tables are the same one (stride 0)
    s = Repeated(cuda_device, dtype, 1, 2, 1, 64, 16, 3, seed=6)
    B, i32 = 65536, dict(dtype=torch.int32, device=cuda_device)
    lens = (torch.arange(B, device=cuda_device) % 41).to(torch.int32)
    new = ((torch.arange(B, device=cuda_device) % 3 > 0) & (lens > 0)).to(torch.int32)
    cu = torch.cat([torch.zeros(1, **i32), torch.cumsum(new, 0).to(torch.int32)])
    n = int(cu[-1])
    g = torch.Generator(device=cuda_device).manual_seed(7)
    Q = torch.randn((n, 2, 64), generator=g, device=cuda_device).to(dtype)
    out, lse = paged.prefix_attention(Q, s.pool_K, s.pool_V, s.table(48)[None].expand(B, 3), lens, cu, return_lse=True)
    k = s.pool_K[:, 0].double().reshape(48, 64)
    v = s.pool_V[:, 0].double().reshape(48, 64)
    score = Q.double() @ k.T * s.scale
    seen = torch.arange(48, device=cuda_device) < lens[new > 0][:, None]
    score = score.masked_fill(~seen[:, None], float("-inf"))
    p = torch.softmax(score, -1)
    want, A = p @ v, p @ v.abs()
    u, e = torch.finfo(dtype).eps / 2, 2.0 ** -24
    top = s.scale * (Q.double().abs() @ k.abs().T).amax(-1)
    per = (0 if dtype == F32 else u) + 2 * (64 + 8) * e * top + 2 * (48 * e + 2.0 ** -21)
    assert ((out.double() - want).abs() <= u * want.abs() + per[..., None] * A).all()
    z = torch.logsumexp(score, -1)
    assert ((lse.double() - z).abs() <= (64 + 8) * e * top + 48 * e + 2.0 ** -21 + 2 * e * z.abs()).all()


def test_block_tables_of_one_very_long_request(cuda_device):
    # 2^26 new tokens and a million blocks of one request, beside a short one
    L, n = 64, (1 << 26) + 5
    F = n // L + 4
    i32 = dict(dtype=torch.int32, device=cuda_device)
    ring = torch.arange(F, **i32).flip(0).contiguous()
    tables = torch.full((2, n // L + 2), -1, **i32)
    t = paged.block_tables(torch.zeros(2, **i32), _dev([n, 3], cuda_device), tables, ring, _dev([7, F], cuda_device),
                           block_len=L, n_tokens=n + 3)
    held = n // L + 1
    taken = ring[(torch.arange(held + 1, device=cuda_device) + 7) % F]
    assert torch.equal(t.tables[0, :held], taken[:held]) and (t.tables[0, held:] == -1).all()
    assert t.tables[1, 0] == taken[held] and (t.tables[1, 1:] == -1).all()
    p = torch.arange(n, device=cuda_device)
    assert torch.equal(t.slot_map[:n].long(), taken[p // L].long() * L + p % L)
    assert t.slot_map[n:].tolist() == [int(taken[held]) * L + i for i in range(3)]
    assert t.lens.tolist() == [n, 3] and t.cu_new.tolist() == [0, n, n + 3] and int(t.n_short) == 0
    assert t.free_state.tolist() == [(7 + held + 1) % F, F - held - 1]
