"""16-bit expert products (grouped_gemm, moe_expert_ffn_w16) against plain 64-bit forms of the same formulas.

Tolerances are bounds on the arithmetic, element by element: an fp32 sum of m products is off by at most
(m + 8) * 2^-23 times the sum of the absolute products (the tensor core may truncate, hence 2^-23 and not 2^-24), a
rounding to 16 bits by half a step (bf16 2^-8, fp16 2^-11 of the value, or 2^-25 below fp16's normal range).  The FFN's
bound on h would hide a mistake of a few percent behind its worst case, so its result is also held to the root mean
square of two independent roundings, each at most half a step / sqrt(3), with a factor 1.5."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
U = 2.0 ** -23


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    return torch.device("cuda:0")


def _randn(shape, dtype, dev, seed, scale=1.0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)


def _i32(v, dev):
    return torch.tensor(np.asarray(v, np.int32), device=dev)


def _offsets(counts, dev):
    return _i32(np.concatenate([[0], np.cumsum(counts)]), dev)


def _grouped_ref(x, w, offs, rows):
    """y, bound on an fp32 sum, and which rows are written."""
    P = rows.numel()
    y = torch.zeros((P, w.shape[1]), dtype=torch.float64, device=x.device)
    b = torch.zeros_like(y)
    written = torch.zeros(P, dtype=torch.bool, device=x.device)
    o = offs.tolist()
    for e in range(w.shape[0]):
        if o[e + 1] <= o[e]:
            continue
        r = rows[o[e]:o[e + 1]].long()
        ok = (r >= 0) & (r < x.shape[0])
        xe = x[r.clamp(0, x.shape[0] - 1)].double()
        we = w[e].double()
        y[o[e]:o[e + 1]] = xe @ we.T
        b[o[e]:o[e + 1]] = xe.abs() @ we.abs().T * ((x.shape[1] + 8) * U)
        written[o[e]:o[e + 1]] = ok
    return y, b, written


def _check(y, ref, bound, what):
    d = (y.double() - ref).abs()
    bad = ~(d <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d - bound).max()):.3e} over the bound"


CASES = [  # counts of every expert, n tokens, K, N
    ([1], 1, 8, 1),
    ([1, 0, 0, 2], 2, 64, 16),
    ([0, 0, 7], 3, 72, 65),
    ([16, 17, 0, 15, 1, 33], 50, 128, 130),
    ([5, 300, 0, 129, 64], 200, 520, 257),
    ([1] * 40, 7, 1024, 512),
    ([3, 0, 1, 9] * 16, 64, 264, 96),
    ([257, 511, 256, 1, 255], 700, 1032, 515),
    ([1100], 1100, 456, 1000),
    ([0, 0, 0], 4, 64, 64),
    ([700, 2, 0, 1400], 900, 2048, 640),
    ([40, 24, 70], 100, 6144, 320),
    ([3], 3, 6144, 200),            # a cluster of blocks per item
    ([2, 0, 5], 9, 2184, 333),
    ([16, 15], 31, 4096, 128),
    ([2], 2, 2056, 70),
    ([30] * 9, 100, 136, 264),      # tiles of 32, 64 and 128 rows
    ([100, 90, 0, 110], 130, 264, 520),
    ([200] * 10, 500, 72, 1111),
    ([255, 257, 512, 3, 300], 640, 200, 2050),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out_f32", [False, True])
def test_grouped_gemm(dev, case, dtype, out_f32):
    from glmserve_b200 import ops
    counts, n, K, N = CASES[case]
    P, pad = int(sum(counts)), 5
    x, w = _randn((n, K), dtype, dev, case), _randn((len(counts), N, K), dtype, dev, 100 + case, 0.05)
    rng = np.random.default_rng(case)
    rows = _i32(rng.integers(0, n, P + pad), dev)
    offs = _offsets(counts, dev)
    od = torch.float32 if out_f32 else dtype
    out = torch.full((P + pad, N), 7.0, dtype=od, device=dev)
    got = ops.grouped_gemm(x, w, offs, rows=rows, out=out)
    assert got is out and ops.operators16_status() == 0
    ref, b, _ = _grouped_ref(x, w, offs, rows)
    _check(out[:P], ref[:P], b[:P] + HALF[od] * ref[:P].abs() * (1 + U) + TINY[od], "grouped_gemm")
    assert bool((out[P:] == 7.0).all()), "rows behind the last segment were written"
    again = ops.grouped_gemm(x, w, offs, rows=rows, out=torch.full_like(out, 7.0))
    assert torch.equal(again, out)


def test_grouped_gemm_without_rows_and_first_segment_not_at_zero(dev):
    from glmserve_b200 import ops
    x, w = _randn((90, 136), torch.bfloat16, dev, 1), _randn((3, 200, 136), torch.bfloat16, dev, 2)
    offs = _i32([4, 30, 30, 77], dev)
    out = torch.full((90, 200), -3.0, dtype=torch.bfloat16, device=dev)
    ops.grouped_gemm(x, w, offs, out=out)
    ref, b, _ = _grouped_ref(x, w, offs, torch.arange(90, device=dev))
    _check(out[4:77], ref[4:77], b[4:77] + HALF[torch.bfloat16] * ref[4:77].abs() * (1 + U), "no rows")
    assert bool((out[:4] == -3).all() and (out[77:] == -3).all())


def test_grouped_gemm_skips_rows_out_of_range(dev):
    from glmserve_b200 import ops
    x, w = _randn((20, 64), torch.float16, dev, 3), _randn((2, 48, 64), torch.float16, dev, 4)
    rows = _i32([0, -1, 19, 20, 5, 2 ** 31 - 1, -2 ** 31, 7], dev)
    offs = _i32([0, 5, 8], dev)
    out = torch.full((8, 48), 9.0, dtype=torch.float16, device=dev)
    ops.grouped_gemm(x, w, offs, rows=rows, out=out)
    ref, b, written = _grouped_ref(x, w, offs, rows)
    assert written.tolist() == [True, False, True, False, True, False, False, True]
    _check(out[written], ref[written], (b + HALF[torch.float16] * ref.abs() * (1 + U) + 2.0 ** -25)[written], "written rows")
    assert bool((out[~written] == 9.0).all())


def test_grouped_gemm_nan_and_inf_stay_in_their_row(dev):
    from glmserve_b200 import ops
    x, w = _randn((40, 200), torch.bfloat16, dev, 5), _randn((2, 70, 200), torch.bfloat16, dev, 6)
    x[3] = float("nan")
    x[11, 199] = float("inf")
    offs = _i32([0, 25, 40], dev)
    clean = x.clone()
    clean[3] = 0
    clean[11] = 0
    y, yc = ops.grouped_gemm(x, w, offs), ops.grouped_gemm(clean, w, offs)
    assert bool(y[3].isnan().all()) and not bool(y[11].isfinite().any())
    keep = [i for i in range(40) if i not in (3, 11)]
    assert torch.equal(y[keep], yc[keep])


def test_grouped_gemm_weights_beyond_two_to_the_31_elements(dev):
    from glmserve_b200 import ops
    E, N, K = 40, 4096, 16384
    w = torch.zeros((E, N, K), dtype=torch.bfloat16, device=dev)
    w[39] = _randn((N, K), torch.bfloat16, dev, 8, 0.02)
    x = _randn((3, K), torch.bfloat16, dev, 9)
    offs = _i32([0] * 39 + [0, 3], dev)
    y = ops.grouped_gemm(x, w, offs, out_dtype=torch.float32)
    ref, b, _ = _grouped_ref(x, w, offs, torch.arange(3, device=dev))
    _check(y, ref, b + HALF[torch.float32] * ref.abs(), "large weights")


def _ffn_ref(x, ids, wt, gate, up, down, dtype):
    n, H = x.shape
    E, I = gate.shape[:2]
    out = torch.zeros((n, H), dtype=torch.float64, device=x.device)
    bound, mag = torch.zeros_like(out), torch.zeros_like(out)
    for e in range(E):
        t, k = (ids == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        xe, w = x[t].double(), wt[t, k].double()[:, None]
        g64, u64, d64 = gate[e].double(), up[e].double(), down[e].double()
        g, u = xe @ g64.T, xe @ u64.T
        h = torch.nn.functional.silu(g) * u
        dg, du = (xe.abs() @ g64.abs().T) * ((H + 8) * U), (xe.abs() @ u64.abs().T) * ((H + 8) * U)
        # |silu'| <= 1.1; silu itself evaluated to 2^-20
        dh = (1.1 * dg * (u.abs() + du) + torch.nn.functional.silu(g).abs() * du) * (1 + U) + (HALF[dtype] + 2.0 ** -20) * h.abs() + TINY[dtype]
        y, ya = h @ d64.T, h.abs() @ d64.abs().T
        dy = dh @ d64.abs().T + ya * ((I + 8) * U)
        out.index_add_(0, t, w * y)
        bound.index_add_(0, t, w.abs() * dy)
        mag.index_add_(0, t, w.abs() * y.abs())
    return out, bound + mag * ((ids.shape[1] + 2) * U)


FFN = [  # n, topk, E, ids below `of`, H, I
    (1, 1, 1, 1, 8, 8),
    (1, 8, 32, 32, 1024, 512),
    (3, 2, 4, 16, 136, 72),
    (17, 4, 16, 16, 256, 128),
    (64, 8, 32, 256, 1024, 264),
    (333, 3, 5, 5, 520, 264),
    (700, 2, 8, 8, 1024, 1032),
    (2500, 4, 6, 6, 264, 136),
    (2, 2, 3, 3, 4096, 200),        # a cluster of blocks per item
    (32, 8, 20, 20, 128, 2304),     # 256 slots, lists made in the kernel
    (100, 2, 3, 3, 264, 520),       # 200 slots, the pair kernel
    (129, 2, 64, 64, 72, 128),      # 258 slots
    (5, 300, 400, 400, 64, 64),     # more slots a token than a block has threads
]


def _ffn_case(case, dtype, dev):
    n, topk, E, of, H, I = FFN[case]
    x = _randn((n, H), dtype, dev, case)
    gate, up = _randn((E, I, H), dtype, dev, 10 + case, 0.05), _randn((E, I, H), dtype, dev, 20 + case, 0.05)
    down = _randn((E, H, I), dtype, dev, 30 + case, 0.05)
    rng = np.random.default_rng(case)
    ids = np.stack([rng.permutation(of)[:topk] for _ in range(n)]).astype(np.int32)
    ids[ids >= E] = [-1, E, 2 ** 31 - 1][case % 3]
    wt = torch.from_numpy((rng.random((n, topk)) + 0.1).astype(np.float32)).to(dev)
    return x, torch.from_numpy(ids).to(dev), wt, gate, up, down


@pytest.mark.parametrize("case", range(len(FFN)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out_f32", [False, True])
def test_expert_ffn(dev, case, dtype, out_f32):
    from glmserve_b200 import ops
    args = _ffn_case(case, dtype, dev)
    od = torch.float32 if out_f32 else dtype
    out = ops.moe_expert_ffn_w16(*args, out_dtype=od)
    assert ops.operators16_status() == 0 and out.dtype == od
    ref, b = _ffn_ref(*args, dtype)
    _check(out, ref, b + HALF[od] * ref.abs() + TINY[od], "ffn")
    if ref.numel() >= 4096:
        rel = float((out.double() - ref).norm() / ref.norm())
        assert rel <= 1.5 * ((HALF[dtype] ** 2 + HALF[od] ** 2) / 3) ** 0.5, rel
    assert torch.equal(ops.moe_expert_ffn_w16(*args, out_dtype=od), out)


def test_expert_ffn_token_without_a_slot_is_zero_and_repeated_expert_counts_twice(dev):
    from glmserve_b200 import ops
    x, ids, wt, gate, up, down = _ffn_case(3, torch.bfloat16, dev)
    ids[0] = -1
    ids[1] = 5
    out = ops.moe_expert_ffn_w16(x, ids, wt, gate, up, down, out=torch.full_like(x, float("nan")))
    assert bool((out[0] == 0).all())
    ref, b = _ffn_ref(x, ids, wt, gate, up, down, torch.bfloat16)
    _check(out, ref, b + HALF[torch.bfloat16] * ref.abs(), "repeated expert")
    none = ops.moe_expert_ffn_w16(x, torch.full_like(ids, -1), wt, gate, up, down)
    assert bool((none == 0).all())


def test_expert_ffn_intermediate_beyond_fp16_saturates(dev):
    from glmserve_b200 import ops
    x = torch.full((1, 64), 100.0, dtype=torch.float16, device=dev)
    gate = torch.full((1, 64, 64), 1.0, dtype=torch.float16, device=dev)
    down = torch.full((1, 64, 64), 2.0 ** -10, dtype=torch.float16, device=dev)
    down[:, :, 1::2] *= -1
    ids, wt = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.ones((1, 1), device=dev)
    out = ops.moe_expert_ffn_w16(x, ids, wt, gate, gate, down)   # h = 6400^2, then sums that cancel
    assert bool((out == 0).all())


def test_router_dispatch_products_and_ffn_together(dev):
    """The operators as a layer uses them: router, dispatch, gate and up products, down product by hand
    against the fused FFN; and the fp32-weight operator on the same values."""
    from glmserve_b200 import ops
    n, E, topk, H, I = 77, 16, 4, 256, 128
    dtype = torch.bfloat16
    x = _randn((n, H), dtype, dev, 1)
    gate, up, down = (_randn(s, dtype, dev, 2 + i, 0.05) for i, s in enumerate([(E, I, H), (E, I, H), (E, H, I)]))
    ids, wt = ops.moe_router(_randn((n, E), torch.float32, dev, 9), None, topk)
    offs, tok, col = ops.moe_dispatch(ids, E)
    g, u = (ops.grouped_gemm(x, m, offs, rows=tok, out_dtype=torch.float32) for m in (gate, up))
    h = (torch.nn.functional.silu(g) * u).to(dtype)
    y = ops.grouped_gemm(h, down, offs, out_dtype=torch.float32)
    by_hand = torch.zeros((n, H), dtype=torch.float64, device=dev)
    by_hand.index_add_(0, tok.long(), wt[tok.long(), col.long()].double()[:, None] * y.double())
    out = ops.moe_expert_ffn_w16(x, ids, wt, gate, up, down, out_dtype=torch.float32)
    ref, b = _ffn_ref(x, ids, wt, gate, up, down, dtype)
    _check(out, ref, b + HALF[torch.float32] * ref.abs(), "fused")
    _check(by_hand, ref, b + HALF[torch.float32] * ref.abs(), "by hand")
    old = ops.moe_expert_ffn(x.float(), ids, wt, gate.float(), up.float(), down.float())
    _check(out, old.double(), 2 * b + 2 * HALF[torch.float32] * ref.abs(), "fp32 operator")


def test_expert16_graph_replay_and_two_streams(dev):
    from glmserve_b200 import ops
    a, b = _ffn_case(4, torch.bfloat16, dev), _ffn_case(6, torch.bfloat16, dev)
    want_a, want_b = ops.moe_expert_ffn_w16(*a), ops.moe_expert_ffn_w16(*b)
    offs, tok, _ = ops.moe_dispatch(b[1], b[3].shape[0])
    want_g = ops.grouped_gemm(b[0], b[3], offs, rows=tok)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        with torch.cuda.stream(s1):
            outs.append((want_a, ops.moe_expert_ffn_w16(*a)))
        with torch.cuda.stream(s2):
            outs.append((want_b, ops.moe_expert_ffn_w16(*b)))
            outs.append((want_g, ops.grouped_gemm(b[0], b[3], offs, rows=tok)))
    torch.cuda.synchronize()
    assert all(torch.equal(w, o) for w, o in outs)
    x = b[0].clone()
    out, y = torch.empty_like(x), torch.empty_like(want_g)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.moe_expert_ffn_w16(x, *b[1:], out=out)
        ops.grouped_gemm(x, b[3], offs, rows=tok, out=y)
    for scale in (1.0, 0.5):
        x.copy_(b[0] * scale)
        out.zero_(), y.zero_()
        graph.replay()
        assert torch.equal(out, ops.moe_expert_ffn_w16(x, *b[1:])) and torch.equal(y, ops.grouped_gemm(x, b[3], offs, rows=tok))
    assert ops.operators16_status() == 0


def test_empty_batches(dev):
    from glmserve_b200 import ops
    x0 = torch.empty((0, 64), dtype=torch.bfloat16, device=dev)
    w = _randn((2, 32, 64), torch.bfloat16, dev, 1)
    offs = _i32([0, 0, 0], dev)
    assert ops.grouped_gemm(x0, w, offs).shape == (0, 32)
    ids, wt = torch.empty((0, 2), dtype=torch.int32, device=dev), torch.empty((0, 2), device=dev)
    assert ops.moe_expert_ffn_w16(x0, ids, wt, w, w, w.transpose(1, 2).contiguous()).shape == (0, 64)


@pytest.mark.parametrize("P", [900, 18000])             # few rows per expert, and many
def test_grouped_gemm_of_1024_experts(dev, P):
    from glmserve_b200 import ops
    rng = np.random.default_rng(P)
    counts = np.bincount(rng.integers(0, 1024, P), minlength=1024)
    counts[-1] += 1                                      # the last expert has a row
    P = int(counts.sum())
    x, w = _randn((300, 72), torch.bfloat16, dev, 5), _randn((1024, 40, 72), torch.bfloat16, dev, 6)
    offs, rows = _offsets(counts, dev), _i32(rng.integers(0, 300, P), dev)
    y = ops.grouped_gemm(x, w, offs, rows=rows, out_dtype=torch.float32)
    ref, b, written = _grouped_ref(x, w, offs, rows)
    assert written.all()
    _check(y, ref, b + HALF[torch.float32] * ref.abs(), "1024 experts")


@pytest.mark.parametrize("n", [32, 100])                 # lists made inside the product, and by the dispatch
def test_expert_ffn_of_1024_experts(dev, n):
    from glmserve_b200 import ops
    E, topk, H, I = 1024, 8, 64, 40
    x, wt = _randn((n, H), torch.bfloat16, dev, 1), _randn((n, topk), torch.float32, dev, 5)
    gate, up = _randn((E, I, H), torch.bfloat16, dev, 2, 0.05), _randn((E, I, H), torch.bfloat16, dev, 3, 0.05)
    down = _randn((E, H, I), torch.bfloat16, dev, 4, 0.05)
    ids = _i32(np.random.default_rng(n).integers(0, E, (n, topk)), dev)
    ids[0, 0] = E - 1
    out = ops.moe_expert_ffn_w16(x, ids, wt, gate, up, down, out_dtype=torch.float32)
    ref, b = _ffn_ref(x, ids, wt, gate, up, down, torch.bfloat16)
    _check(out, ref, b + HALF[torch.float32] * ref.abs(), "1024 experts")


@pytest.mark.parametrize("K,N,P", [(64, 130, 40), (4096, 64, 12), (264, 520, 300)])     # few rows, a cluster per item, many rows
def test_grouped_gemm_bad_offsets_stay_inside(dev, K, N, P):
    from glmserve_b200 import ops
    x, w = _randn((P, K), torch.bfloat16, dev, 1), _randn((3, N, K), torch.bfloat16, dev, 2)
    for rows in (None, torch.arange(P, dtype=torch.int32, device=dev)):
        y = torch.full((P, N), 7.0, dtype=torch.bfloat16, device=dev)
        ops.grouped_gemm(x, w, _i32([0, P, P // 2, P], dev), rows=rows, out=y)          # descends: nothing is written
        assert bool((y == 7).all())
        ops.grouped_gemm(x, w, _i32([-9, 2, 2, 2 ** 31 - 1], dev), rows=rows, out=y)    # clamped to [0, P]
        want = ops.grouped_gemm(x, w, _i32([0, 2, 2, P], dev), rows=rows)
        assert torch.equal(y, want)
    assert ops.operators16_status() == 0


def test_calls_of_different_kernels_follow_each_other(dev):
    """Every kernel's launch may begin while the one ahead ends: 16-bit and int4 operators, small and large, in turn."""
    from glmserve_b200 import ops
    a, b, c = (_ffn_case(i, torch.bfloat16, dev) for i in (1, 6, 8))
    offs, tok, _ = ops.moe_dispatch(b[1], b[3].shape[0])
    one, three = ops.moe_expert_ffn_w16(*a), ops.moe_expert_ffn_w16(*c)
    two, rows = ops.moe_expert_ffn_w16(*b), ops.grouped_gemm(b[0], b[3], offs, rows=tok)
    x = a[0].clone()
    torch.cuda.synchronize()
    for _ in range(20):
        x.zero_()
        x.copy_(a[0])
        got = [ops.moe_expert_ffn_w16(x, *a[1:]), ops.moe_expert_ffn_w16(*c)]
        x.zero_()                                        # after its last reader
        o2, t2, _ = ops.moe_dispatch(b[1], b[3].shape[0])
        got += [ops.grouped_gemm(b[0], b[3], o2, rows=t2), ops.moe_expert_ffn_w16(*b), ops.moe_expert_ffn_w16(*c)]
        assert all(torch.equal(g, w) for g, w in zip(got, (one, three, rows, two, three)))


# few rows per expert, a cluster of blocks per item, many rows per expert; and lists of more than 256 slots
NONFINITE = [(4, 2, 4, 136, 72), (2, 2, 3, 4096, 200), (100, 2, 3, 264, 520), (150, 2, 3, 264, 520), (70, 4, 64, 136, 72)]


@pytest.mark.parametrize("shape", NONFINITE)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_expert_ffn_nan_and_infinite_tokens_stay_in_their_row(dev, shape, dtype):
    """A NaN reaches every gate sum of its token; an infinity makes gate sums of both signs, and silu(-inf) is NaN."""
    from glmserve_b200 import ops
    n, topk, E, H, I = shape
    x = _randn((n, H), dtype, dev, 1)
    gate, up, down = (_randn(s, dtype, dev, 2 + i, 0.05) for i, s in enumerate([(E, I, H), (E, I, H), (E, H, I)]))
    rng = np.random.default_rng(n)
    ids = _i32(np.stack([rng.permutation(E)[:topk] for _ in range(n)]), dev)
    wt = torch.from_numpy((rng.random((n, topk)) + 0.1).astype(np.float32)).to(dev)
    clean = ops.moe_expert_ffn_w16(x, ids, wt, gate, up, down)
    for bad, value in ((n - 1, float("nan")), (n // 2, float("inf")), (0, -float("inf"))):
        y = x.clone()
        y[bad, H - 3] = value
        out = ops.moe_expert_ffn_w16(y, ids, wt, gate, up, down)
        assert bool(out[bad].isnan().all()), value
        keep = [t for t in range(n) if t != bad]
        assert torch.equal(out[keep], clean[keep])
    assert bool(clean.isfinite().all())


@pytest.mark.parametrize("shape", NONFINITE)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_expert_ffn_infinity_goes_through(dev, shape, dtype):
    """Positive weights: an infinite activation gives an infinite gate, an infinite h and an infinite result."""
    from glmserve_b200 import ops
    n, topk, E, H, I = shape
    x = _randn((n, H), dtype, dev, 1)
    gate, up, down = (_randn(s, dtype, dev, 2 + i, 0.05).abs() + 0.01 for i, s in enumerate([(E, I, H), (E, I, H), (E, H, I)]))
    ids = _i32(np.stack([np.random.default_rng(t).permutation(E)[:topk] for t in range(n)]), dev)
    x[n // 2, 1] = float("inf")
    out = ops.moe_expert_ffn_w16(x, ids, torch.ones((n, topk), device=dev), gate, up, down, out_dtype=torch.float32)
    want = torch.zeros_like(out, dtype=torch.bool)
    want[n // 2] = True
    assert torch.equal(out == float("inf"), want) and not bool(out.isnan().any())


def test_expert_ffn_of_more_features_than_a_grid_has_blocks_for(dev):
    """65535 blocks of 1024 features and a ragged rest, one token; x has few values, so that 64-bit sums are quick."""
    from glmserve_b200 import ops
    H, I, dtype = 65535 * 1024 + 2056, 8, torch.bfloat16
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    x = torch.zeros((1, H), dtype=dtype, device=dev)
    at = torch.cat([torch.randint(H, (62,), generator=g, device=dev), torch.tensor([0, H - 1], device=dev)])
    x[0, at] = torch.randn(64, generator=g, device=dev).to(dtype)
    gate, up, down = (torch.empty(s, dtype=dtype, device=dev).normal_(0, 0.05, generator=g) for s in ((1, I, H), (1, I, H), (1, H, I)))
    ids, wt = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.full((1, 1), 0.75, device=dev)
    out = ops.moe_expert_ffn_w16(x, ids, wt, gate, up, down, out=torch.full((1, H), float("nan"), device=dev))
    assert ops.operators16_status() == 0
    at = at.unique()
    xs = x[0, at].double()
    gs, us = gate[0][:, at].double(), up[0][:, at].double()
    g64, u64 = gs @ xs, us @ xs
    h = torch.nn.functional.silu(g64) * u64
    # sums of 64 products: the zeros beside them add nothing
    dg, du = gs.abs() @ xs.abs() * (72 * U), us.abs() @ xs.abs() * (72 * U)
    dh = (1.1 * dg * (u64.abs() + du) + torch.nn.functional.silu(g64).abs() * du) * (1 + U) + (HALF[dtype] + 2.0 ** -20) * h.abs()
    for a in range(0, H, 1 << 24):
        d = down[0, a:a + (1 << 24)].double()
        ref, mag = 0.75 * (d @ h), d.abs() @ h.abs()
        _check(out[0, a:a + (1 << 24)], ref, 0.75 * (d.abs() @ dh) + mag * (20 * U), f"features from {a}")


def _sparse(n, K, at, dev, seed):
    """[n, K] of zeros but for the columns `at`, made without a dense copy in another type."""
    x = torch.zeros((n, K), dtype=torch.bfloat16, device=dev)
    x[:, at] = _randn((n, at.numel()), torch.bfloat16, dev, seed)
    return x


@pytest.mark.parametrize("E,P,K", [(38, 38, 1 << 29), (1, 17, 1 << 30)])     # few rows per expert, and many
def test_grouped_gemm_sum_that_takes_a_second(dev, E, P, K):
    """One block (pair) after the other takes over 2^23 steps along K: its waits must last as long as the sum does."""
    from glmserve_b200 import ops
    at = torch.tensor([0, 5, 70, K // 3, K // 2, K - 65, K - 2, K - 1], device=dev)
    x, w = _sparse(P if E == 1 else 1, K, at, dev, 1), _sparse(E, K, at, dev, 2)
    rows = None if E == 1 else torch.zeros(P, dtype=torch.int32, device=dev)
    y = ops.grouped_gemm(x, w[:, None], _i32(np.arange(E + 1) * (P // E), dev), rows=rows, out=torch.full((P, 1), float("nan"), device=dev))
    assert ops.operators16_status() == 0
    xs, ws = x[:, at].double(), w[:, at].double()
    # sums of eight products: the zeros beside them add nothing
    ref, mag = (xs @ ws.T, xs.abs() @ ws.abs().T) if E == 1 else (ws @ xs.T, ws.abs() @ xs.abs().T)
    _check(y, ref, mag * (16 * U), "long sum")
    del x, w, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("case", [1, 5, 8, 10])          # lists in the kernel, the pair kernel, a cluster, few slots
def test_expert_ffn_in_place(dev, case):
    from glmserve_b200 import ops
    x, *rest = _ffn_case(case, torch.bfloat16, dev)
    want = ops.moe_expert_ffn_w16(x, *rest)
    assert ops.moe_expert_ffn_w16(x, *rest, out=x) is x and torch.equal(x, want)
