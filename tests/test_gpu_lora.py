"""Low-rank adapters (lora_add) against a plain 64-bit form.  Bounds as in test_gpu_expert16.py: an fp32 sum of m
products is off by (m + 8) * 2^-23 of the sum of absolute products; B is applied to the fp32 values A x in pieces
that keep at least 21 bits (2^-21 of every product); y is rounded once."""
import numpy as np
import pytest

from test_gpu_expert16 import HALF, TINY, U, _check, _i32, _randn
from test_gpu_expert16 import _sparse

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _ref(y0, x, A, B, offs, rows, ranks, scales):
    y = y0.double().clone()
    bound = torch.zeros_like(y)
    o = offs.tolist()
    for a in range(A.shape[0]):
        t = rows[o[a]:o[a + 1]].long()
        t = t[(t >= 0) & (t < x.shape[0])]
        if not t.numel():
            continue
        r = int(ranks[a]) if ranks is not None else A.shape[1]
        s = float(scales[a]) if scales is not None else 1.0
        xa, Aa, Ba = x[t].double(), A[a, :r].double(), B[a, :, :r].double()
        v, va = s * (xa @ Aa.T), abs(s) * (xa.abs() @ Aa.abs().T)
        d, da = v @ Ba.T, v.abs() @ Ba.abs().T
        y[t] += d
        bound[t] = va @ Ba.abs().T * ((x.shape[1] + 10) * U) + da * ((r + 8) * U + 2.0 ** -21) + (y0[t].double().abs() + d.abs()) * U
    return y, bound


CASES = [  # n, K, N, adapters, R, ranks, share without an adapter
    (1, 8, 1, 1, 1, None, 0.0),
    (1, 1024, 1024, 8, 16, None, 0.0),
    (3, 72, 65, 2, 5, "mixed", 0.4),
    (64, 512, 520, 64, 16, None, 0.1),
    (64, 6144, 640, 7, 16, None, 0.0),
    (100, 264, 1030, 3, 24, "mixed", 0.3),
    (517, 1032, 2050, 21, 33, "mixed", 0.3),
    (1030, 128, 136, 4, 64, None, 0.0),
    (300, 2048, 300, 2, 256, "mixed", 0.2),
    (2000, 256, 264, 1000, 8, "zeros", 0.5),
    (700, 520, 1024, 5, 128, "mixed", 1.0),
    (40, 16, 6144, 2, 7, None, 0.0),
    (3, 4104, 1032, 4, 32, "mixed", 0.0),       # one launch
    (190, 264, 520, 1, 16, None, 0.0),
    (100, 512, 264, 50, 64, "mixed", 0.1),      # 8-row tiles, 16-row tiles
    (1100, 136, 264, 4, 16, "mixed", 0.1),      # 32-row tiles
    (1300, 72, 130, 4, 60, "mixed", 0.1),
    (1300, 264, 5300, 3, 64, "mixed", 0.1),     # tcgen05
    (4500, 72, 5900, 9, 32, "zeros", 0.2),
    (1210, 64, 5260, 40, 40, None, 0.0),
    (1050, 128, 200, 3, 200, "mixed", 0.0),
    (1300, 72, 2055, 3, 33, "mixed", 0.1),      # tcgen05, B laid out by hand
    (700, 72, 3941, 5, 7, None, 0.1),
    (600, 136, 4501, 2, 61, "zeros", 0.0),
]


def _case(i, dtype, ydt, dev):
    n, K, N, nA, R, ranks, bare = CASES[i]
    rng = np.random.default_rng(i)
    ids = rng.integers(0, nA, n).astype(np.int32)
    ids[rng.random(n) < bare] = -1
    x, A, B = _randn((n, K), dtype, dev, i), _randn((nA, R, K), dtype, dev, 40 + i, 0.05), _randn((nA, N, R), dtype, dev, 80 + i, 0.05)
    rk = None
    if ranks:
        rk = rng.integers(0 if ranks == "zeros" else 1, R + 1, nA).astype(np.int32)
        for a in range(nA):    # what lies behind a rank must not matter
            A[a, rk[a]:] = float("nan")
            B[a, :, rk[a]:] = float("nan")
        rk = torch.from_numpy(rk).to(dev)
    scales = torch.from_numpy(rng.uniform(0.5, 2.0, nA).astype(np.float32)).to(dev) if i % 2 else None
    return _randn((n, N), ydt, dev, 120 + i), x, A, B, torch.from_numpy(ids).to(dev), rk, scales


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("y_f32", [True, False])
def test_lora_add(dev, case, dtype, y_f32):
    from glmserve_b200 import ops
    ydt = torch.float32 if y_f32 else dtype
    y0, x, A, B, ids, ranks, scales = _case(case, dtype, ydt, dev)
    offs, rows, _ = ops.moe_dispatch(ids[:, None].contiguous(), A.shape[0])
    y = y0.clone()
    assert ops.lora_add(y, x, A, B, offs, rows, ranks=ranks, scales=scales) is y
    ref, b = _ref(y0, x, A, B, offs, rows, ranks, scales)
    _check(y, ref, b + HALF[ydt] * (ref.abs() + b) + TINY[ydt], "lora")
    assert torch.equal(y[ids < 0], y0[ids < 0])
    again = y0.clone()
    assert torch.equal(ops.lora_add(again, x, A, B, offs, rows, ranks=ranks, scales=scales), y)


def test_lora_rows_out_of_range_are_skipped(dev):
    from glmserve_b200 import ops
    y0, x, A, B, _, _, _ = _case(3, torch.bfloat16, torch.float32, dev)
    rows = _i32([5, -1, 64, 2 ** 31 - 1, 9, 0], dev)
    offs = _i32([0] * 10 + [4] + [6] * 54, dev)
    y = ops.lora_add(y0.clone(), x, A, B, offs, rows)
    ref, b = _ref(y0, x, A, B, offs, rows, None, None)
    _check(y, ref, b + HALF[torch.float32] * (ref.abs() + b), "lora")
    keep = [i for i in range(64) if i not in (5, 9, 0)]
    assert torch.equal(y[keep], y0[keep])


def test_lora_beside_the_int4_projection(dev):
    """gemm_w4a16 and the adapters of a mixed batch, as a projection with adapters runs."""
    import oracle
    from glmserve_b200 import ops
    from glmserve_b200.quant import quantize_w4_np
    rng = np.random.default_rng(0)
    n, K, N, nA, R = 9, 256, 192, 3, 8
    q, sc = quantize_w4_np((rng.standard_normal((N, K)) * 0.02).astype(np.float32), 128)
    x = _randn((n, K), torch.bfloat16, dev, 1)
    A, B = _randn((nA, R, K), torch.bfloat16, dev, 2, 0.05), _randn((nA, N, R), torch.bfloat16, dev, 3, 0.05)
    ids = _i32([0, 2, -1, 1, 2, 2, -1, 0, 1], dev)
    offs, rows, _ = ops.moe_dispatch(ids[:, None].contiguous(), nA)
    base = ops.gemm_w4a16(x.float(), torch.from_numpy(q).to(dev), torch.from_numpy(sc).to(dev), 128)
    np.testing.assert_allclose(base.cpu().numpy(), oracle.gemm_w4a16(x.float().cpu().numpy(), q, sc, 128), rtol=0, atol=1e-4)
    y = ops.lora_add(base.clone(), x, A, B, offs, rows)
    ref, b = _ref(base, x, A, B, offs, rows, None, None)
    _check(y, ref, b + HALF[torch.float32] * (ref.abs() + b), "projection with adapters")


def test_lora_graph_replay_with_another_batch_and_two_streams(dev):
    from glmserve_b200 import ops
    y0, x, A, B, ids, ranks, scales = _case(6, torch.float16, torch.float32, dev)
    offs, rows, _ = ops.moe_dispatch(ids[:, None].contiguous(), A.shape[0])
    want = ops.lora_add(y0.clone(), x, A, B, offs, rows, ranks=ranks, scales=scales)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                got.append(ops.lora_add(y0.clone(), x, A, B, offs, rows, ranks=ranks, scales=scales))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    y = y0.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.lora_add(y, x, A, B, offs, rows, ranks=ranks, scales=scales)
    y.copy_(y0)
    graph.replay()
    assert torch.equal(y, want)
    other = torch.roll(ids, 7).contiguous()          # the same graph serves the next batch's lists
    o2, r2, _ = ops.moe_dispatch(other[:, None].contiguous(), A.shape[0])
    m = int(o2[-1])
    offs.copy_(o2), rows[:m].copy_(r2[:m]), y.copy_(y0)
    graph.replay()
    ref, b = _ref(y0, x, A, B, o2, r2[:m], ranks, scales)
    _check(y, ref, b + HALF[torch.float32] * (ref.abs() + b), "replayed")


def test_lora_empty_lists(dev):
    from glmserve_b200 import ops
    y0, x, A, B, ids, _, _ = _case(3, torch.bfloat16, torch.float32, dev)
    offs, rows, _ = ops.moe_dispatch(torch.full_like(ids, -1)[:, None].contiguous(), A.shape[0])
    assert torch.equal(ops.lora_add(y0.clone(), x, A, B, offs, rows), y0)
    assert torch.equal(ops.lora_add(y0.clone(), x, A, B, offs, rows[:0]), y0)


def test_lora_of_1024_adapters(dev):
    from glmserve_b200 import ops
    for n in (1, 900, 9000):
        x, A, B = _randn((n, 64), torch.bfloat16, dev, n), _randn((1024, 8, 64), torch.bfloat16, dev, 2, 0.1), _randn((1024, 40, 8), torch.bfloat16, dev, 3)
        ids = _i32(np.random.default_rng(n).integers(0, 1024, n), dev)
        ids[0] = 1023
        offs, rows, _ = ops.moe_dispatch(ids[:, None].contiguous(), 1024)
        y0 = _randn((n, 40), torch.float32, dev, 4)
        y = ops.lora_add(y0.clone(), x, A, B, offs, rows)
        ref, b = _ref(y0, x, A, B, offs, rows, None, None)
        _check(y, ref, b + HALF[torch.float32] * (ref.abs() + b), "1024 adapters")


SHAPES = [1, 6, 14, 15, 17, 21]       # one launch; two of each kind; tcgen05 with and without TMA


@pytest.mark.parametrize("case", SHAPES + [3, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lora_nan_and_infinity_stay_in_their_row(dev, case, dtype):
    from glmserve_b200 import ops
    y0, x, A, B, ids, ranks, scales = _case(case, dtype, torch.float32, dev)
    n = x.shape[0]
    offs, rows, _ = ops.moe_dispatch(ids[:, None].contiguous(), A.shape[0])
    want = ops.lora_add(y0.clone(), x, A, B, offs, rows, ranks=ranks, scales=scales)
    bad = sorted({n // 2, n // 3})
    for i, t in enumerate(bad):
        x[t, i] = [float("nan"), float("inf")][i % 2]
    y = ops.lora_add(y0.clone(), x, A, B, offs, rows, ranks=ranks, scales=scales)
    keep = torch.ones(n, dtype=torch.bool, device=dev)
    keep[bad] = False
    assert torch.equal(y[keep], want[keep])
    for t in bad:
        if int(ids[t]) >= 0 and (ranks is None or int(ranks[int(ids[t])]) > 0):
            assert not bool(torch.isfinite(y[t]).any())


@pytest.mark.parametrize("case", SHAPES)
@pytest.mark.parametrize("big", [3000.0, 2.0 ** -14])
def test_lora_products_outside_fp16(dev, case, big):
    """A x far beyond 65504, or below fp16's normal range, beside fp16 weights: it is never a 16-bit number by itself."""
    from glmserve_b200 import ops
    y0, x, A, B, ids, ranks, scales = _case(case, torch.float16, torch.float32, dev)
    y0, x, A, B = y0 * 0, (x * big).clamp(-60000, 60000), A * (20.0 if big > 1 else 2.0 ** -6), B * 0.125
    offs, rows, _ = ops.moe_dispatch(ids[:, None].contiguous(), A.shape[0])
    y = ops.lora_add(y0.clone(), x, A, B, offs, rows, ranks=ranks, scales=scales)
    ref, b = _ref(y0, x, A, B, offs, rows, ranks, scales)
    assert bool(torch.isfinite(y).all())
    _check(y, ref, b + HALF[torch.float32] * (ref.abs() + b), "scaled")


@pytest.mark.parametrize("case", SHAPES)
def test_lora_bad_offsets_stay_inside(dev, case):
    from glmserve_b200 import ops
    y0, x, A, B, ids, _, _ = _case(case, torch.bfloat16, torch.float32, dev)
    A, B = torch.nan_to_num(A), torch.nan_to_num(B)
    nA, n = A.shape[0], x.shape[0]
    rows = torch.arange(n, dtype=torch.int32, device=dev)
    y = y0.clone()
    ops.lora_add(y, x, A, B, _i32([0, n, n - 1] + [n] * (nA - 2), dev), rows)          # descends: nothing is written
    assert torch.equal(y, y0)
    ops.lora_add(y, x, A, B, _i32([-5] + [0] * (nA - 1) + [2 ** 31 - 1], dev), rows)    # clamped to [0, P]
    assert torch.equal(y, ops.lora_add(y0.clone(), x, A, B, _i32([0] * nA + [n], dev), rows))


@pytest.mark.parametrize("case", SHAPES + [8, 19])      # and ranks whose B is loaded in turn, tcgen05 at rank 40
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lora_small_ranks_beside_large_ones(dev, case, dtype):
    """Odd ranks of A are 2^-36 of the even ones, and half of the features of B read the odd ranks alone: what is small
    in a row of A x keeps its bits beside the row's largest."""
    from glmserve_b200 import ops
    y0, x, A, B, ids, ranks, scales = _case(case, dtype, torch.float32, dev)
    y0 = y0 * 0
    big, small = (_randn(A.shape, torch.float32, dev, s) for s in (500 + case, 600 + case))
    new = (big * 2.0 ** 15).clamp(-60000, 60000)
    new[:, 1::2] = ((small[:, 1::2] * 8).round() * 2.0 ** -24)
    A = torch.where(A.isnan(), A, new.to(dtype))
    new = _randn(B.shape, torch.float32, dev, 700 + case) * 2.0 ** 12
    new[:, :, 0::2] *= 2.0 ** -26
    new[:, 1::2, 0::2] = 0
    B = torch.where(B.isnan(), B, new.to(dtype))
    offs, rows, _ = ops.moe_dispatch(ids[:, None].contiguous(), A.shape[0])
    y = ops.lora_add(y0.clone(), x, A, B, offs, rows, ranks=ranks, scales=scales)
    ref, b = _ref(y0, x, A, B, offs, rows, ranks, scales)
    _check(y, ref, b + HALF[torch.float32] * (ref.abs() + b), "small ranks")


@pytest.mark.parametrize("case", SHAPES + [8, 19])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lora_infinite_entry_beside_large_ones(dev, case, dtype):
    """One rank of A x is infinite, the others are finite beyond 65504: y is infinity of the sign of that rank's B."""
    from glmserve_b200 import ops
    y0, x, A, B, ids, _, _ = _case(case, dtype, torch.float32, dev)
    x, A, B = x.abs() + 1, A.nan_to_num().abs() * 20 + 1000, B.nan_to_num()
    if A.shape[1] < 2:
        pytest.skip("one rank")
    B = torch.where(B.abs() < 0.01, torch.full_like(B, 0.01), B)
    A[:, 0, 0] = float("inf")
    offs, rows, _ = ops.moe_dispatch(ids[:, None].contiguous(), A.shape[0])
    y = ops.lora_add(y0.clone(), x, A, B, offs, rows)
    on = ids >= 0
    want = torch.copysign(torch.full_like(y0, float("inf")), B[ids.clamp(min=0).long(), :, 0].float())
    assert torch.equal(y[on], want[on]) and torch.equal(y[~on], y0[~on])


@pytest.mark.parametrize("case", [0, 3, 14, 15, 17, 21])
def test_lora_products_next_to_the_largest_fp32(dev, case):
    """A x between the largest bf16 number and the largest fp32 number is finite, and so is B A x."""
    from glmserve_b200 import ops
    y0, x, A, B, ids, _, _ = _case(case, torch.bfloat16, torch.float32, dev)
    y0, x, A, B = (torch.zeros_like(t) for t in (y0, x, A, B))
    x[:, 0], x[:, 1] = (2 - 2.0 ** -7) * 2.0 ** 127, 1.25 * 2.0 ** 119
    A[:, 0, :2] = 1
    B[:, :, 0] = 2.0 ** -10
    offs, rows, _ = ops.moe_dispatch(ids[:, None].contiguous(), A.shape[0])
    y = ops.lora_add(y0.clone(), x, A, B, offs, rows)
    value = ((2 - 2.0 ** -7) * 2.0 ** 127 + 1.25 * 2.0 ** 119) * 2.0 ** -10      # exact in fp32
    assert torch.equal(y, torch.where(ids[:, None] >= 0, torch.full_like(y0, value), y0))


@pytest.mark.parametrize("R", [8, 7])            # B by TMA, and laid out by hand
def test_lora_long_sum(dev, R):
    """The second launch starts early and waits for the first, whose eight blocks take 2^21 steps along K each."""
    from glmserve_b200 import ops
    n, K, N = 17, 1 << 30, 160001
    at = torch.tensor([0, 5, 70, K // 3, K // 2, K - 65, K - 2, K - 1], device=dev)
    x, A, B = _sparse(n, K, at, dev, 1), _sparse(R, K, at, dev, 2), _randn((1, N, R), torch.bfloat16, dev, 3)
    y = ops.lora_add(torch.zeros((n, N), device=dev), x, A[None], B, _i32([0, n], dev), torch.arange(n, dtype=torch.int32, device=dev))
    assert ops.operators16_status() == 0
    xs, As, Bs = x[:, at].double(), A[:, at].double(), B[0].double()
    v, va = xs @ As.T, xs.abs() @ As.abs().T
    # sums of eight products and of R: the zeros beside them add nothing
    ref, mag = v @ Bs.T, va @ Bs.abs().T
    _check(y, ref, mag * (18 * U) + v.abs() @ Bs.abs().T * ((R + 8) * U + 2.0 ** -21) + HALF[torch.float32] * ref.abs(), "long sum")
    del x, A, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,nA,R", [(40, 20, 16), (120, 2, 32), (700, 5, 24)])      # one launch, and two
def test_lists_made_right_before_the_call(dev, n, nA, R):
    """The dispatch lets the next kernel start early: every call must see the lists, x and y as they are at its place in
    the stream, while the same buffers are rewritten between the calls."""
    from glmserve_b200 import ops
    rng = np.random.default_rng(n)
    K, N = 264, 520
    A, B = _randn((nA, R, K), torch.bfloat16, dev, 1, 0.1), _randn((nA, N, R), torch.bfloat16, dev, 2)
    ids = [_i32(rng.integers(-1, nA, n), dev)[:, None].contiguous() for _ in range(6)]
    xs = [_randn((n, K), torch.bfloat16, dev, 3 + i) for i in range(6)]
    want = []
    for i, x in zip(ids, xs):
        offs, rows, _ = ops.moe_dispatch(i, nA)
        torch.cuda.synchronize()
        y = ops.lora_add(torch.zeros((n, N), device=dev), x, A, B, offs, rows)
        g = ops.grouped_gemm(x, A, offs, rows=rows, out=torch.zeros((n, R), dtype=torch.bfloat16, device=dev))
        torch.cuda.synchronize()
        want.append((y, g))
    x, cur = torch.empty_like(xs[0]), torch.empty_like(ids[0])
    got = []
    for _ in range(10):
        for i in range(6):
            x.copy_(xs[i]), cur.copy_(ids[i])
            y, g = torch.zeros((n, N), device=dev), torch.zeros((n, R), dtype=torch.bfloat16, device=dev)
            offs, rows, _ = ops.moe_dispatch(cur, nA)
            ops.lora_add(y, x, A, B, offs, rows)
            offs, rows, _ = ops.moe_dispatch(cur, nA)
            ops.grouped_gemm(x, A, offs, rows=rows, out=g)
            got.append((i, y, g))
    assert all(torch.equal(y, want[i][0]) and torch.equal(g, want[i][1]) for i, y, g in got)
