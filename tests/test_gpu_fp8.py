"""Block-scaled 8-bit operators through the C ABI against the 64-bit oracle.  The quantiser is compared bit
for bit; products within a bound that the oracle derives for fp32 sums of the matrix instruction's group sums
(and for 8-bit rounding borders that such a sum can lie next to), plus half a step of the output type."""
import math

import pytest
import torch

from oracle import ref_fp8
from sparse_amd import _lib, fp8, ops

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]
ALL = HALF + [torch.float32]


def within(got, want, bound, dtype):
    tol = bound + ref_fp8.half_step(dtype, want.abs() + bound)
    err = (got.double().cpu() - want).abs()
    assert bool(torch.isfinite(got).all())
    worst = float((err - tol).max())
    assert worst <= 0, f"off by {worst} more than allowed; largest error {float(err.max())}"


def grouped(T):
    """Calls of one or two rows add products in fp32, larger ones in the 8-bit instruction's groups."""
    return T > 2


@pytest.fixture(params=["stream", "tiles"])
def path(request):
    """Both families of kernels, whatever the size would choose."""
    lib = _lib.load()
    before = lib.sparse_hip_fp8_path({"stream": 1, "tiles": 2}[request.param])
    yield request.param
    lib.sparse_hip_fp8_path(before)


def grouped_gate_up(T, path):
    """Only the tiles take gate and up projections in the 8-bit instruction."""
    return T > 2 and path == "tiles"


def rand_rows(T, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 17 * T + K)
    loud = torch.exp(torch.randn(K, generator=g))
    return (torch.randn(T, K, generator=g) * loud).to(dtype)


def rand_weight(N, K, seed=0, pow2=False):
    g = torch.Generator().manual_seed(seed + 31 * N + K)
    nb, kb = fp8.blocks(N), fp8.blocks(K)
    q = (torch.randn(N, K, generator=g) * 100).clamp(-448, 448).to(fp8.E4M3)
    s = torch.exp(torch.randn(nb, kb, generator=g)) * 2e-3
    return q, torch.exp2(torch.round(torch.log2(s))) if pow2 else s


# ------------------------------------------------------------------------------------- quantiser
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("T,K", [(1, 1), (1, 127), (3, 128), (5, 129), (33, 1400), (257, 2048), (2, 8), (40, 1001)])
def test_quantize_is_exact(device, dtype, T, K):
    x = rand_rows(T, K, dtype)
    rows = fp8.quantize(x.to(device))
    q, s = ref_fp8.quantize(x)
    assert torch.equal(rows.values.cpu().double(), q)
    assert torch.equal(rows.scales.cpu().view(torch.uint8).int(), (s + 127).int())
    assert not bool(rows.data[:, K:].view(torch.uint8).any()), "the padding must be zero"
    assert torch.equal(rows.dequantize(torch.float64).cpu(), ref_fp8.rows(x))


def test_quantize_borders(device):
    """Runs whose largest value sits on and beside 448 * 2^s, ties between 8-bit neighbours, subnormals, zeros,
    the smallest and largest fp32 numbers, infinities (which become NaN)."""
    tops = [448.0, 448.0 * (1 + 2 ** -23), 449.0, 447.9, 1.75, 1.7500001, 2.0, 1.0, 2.0 ** -119, 448 * 2.0 ** -120,
            448 * 2.0 ** -121, 2.0 ** -126, 2.0 ** -149, 0.0, 3.0e38, torch.finfo(torch.float32).max]
    x = torch.zeros(len(tops), 256)
    for i, t in enumerate(tops):
        x[i, :128] = torch.linspace(-1, 1, 128) * t
        x[i, 127] = t
        x[i, 128:] = t * torch.tensor([(1 + (2 * j + 1) / 16) * 2.0 ** -(j % 12) / 2 for j in range(128)]) / 9
    q, s = ref_fp8.quantize(x)
    rows = fp8.quantize(x.to(device))
    assert torch.equal(rows.scales.cpu().view(torch.uint8).int(), (s + 127).int())
    got = rows.values.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(q))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(q))


@pytest.mark.parametrize("dtype", ALL)
def test_quantize_non_finite(device, dtype):
    x = rand_rows(4, 300, dtype)
    x[0, 5], x[0, 200], x[1, 0], x[2, :128] = math.nan, math.inf, -math.inf, math.nan
    rows = fp8.quantize(x.to(device))
    q, s = ref_fp8.quantize(x)
    got = rows.values.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(q))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(q))
    assert torch.equal(rows.scales.cpu().view(torch.uint8).int(), (s + 127).int())


def test_quantize_unaligned_rows(device):
    """Rows that start on odd addresses (a view into a larger buffer) give the same bytes."""
    x = rand_rows(3, 256, torch.bfloat16)
    buf = torch.empty(3 * 256 + 1, dtype=torch.bfloat16, device=device)
    view = buf[1:].view(3, 256)
    view.copy_(x)
    a, b = fp8.quantize(view), fp8.quantize(x.to(device))
    assert torch.equal(a.data.view(torch.uint8), b.data.view(torch.uint8))
    assert torch.equal(a.scales.view(torch.uint8), b.scales.view(torch.uint8))


def test_quantize_weight_is_the_quantisers_rule(device):
    w = torch.randn(200, 300, generator=torch.Generator().manual_seed(1)) * 0.02
    w[128:, 256:] = 0
    q, s = fp8.quantize_weight(w)
    for i in range(2):
        for k in range(3):
            b = w[i * 128:(i + 1) * 128, k * 128:(k + 1) * 128].double()
            e = int(ref_fp8.exponent(b.abs().max()))
            assert float(s[i, k]) == 2.0 ** e
            assert torch.equal(q[i * 128:(i + 1) * 128, k * 128:(k + 1) * 128].double(), ref_fp8.round_e4m3(b / 2.0 ** e))
    on_gpu = fp8.quantize_weight(w.to(device))
    assert torch.equal(on_gpu[0].cpu().view(torch.uint8), q.view(torch.uint8)) and torch.equal(on_gpu[1].cpu(), s)


# ---------------------------------------------------------------------------------------- linear
SIZES = [(1, 128, 16), (1, 1, 1), (2, 64, 17), (15, 130, 100), (16, 127, 130), (17, 1000, 33), (31, 384, 256),
         (33, 256, 300), (65, 257, 129), (100, 1400, 64), (129, 128, 257), (300, 500, 520)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("T,K,N", SIZES)
def test_linear(path, device, dtype, T, K, N):
    for pow2 in (False, True):
        x, (q, s) = rand_rows(T, K, dtype), rand_weight(N, K, pow2=pow2)
        w = fp8.Weight.from_quantized(q.to(device), s.to(device))
        want, bound = ref_fp8.product(ref_fp8.rows(x), (q, s), grouped(T))
        x = x.to(device)
        y = fp8.linear(x, w)
        assert y.dtype == dtype
        within(y, want, bound, dtype)
        assert torch.equal(fp8.linear(fp8.quantize(x), w), y), "rows quantised before or inside the call"
        assert torch.equal(w.dequantize(torch.float64).cpu(), ref_fp8.weight(q, s))


@pytest.mark.parametrize("T", [1, 7, 40])
def test_linear_far_from_one(path, device, T):
    """Rows near both ends of the range, runs whose scale is the lowest."""
    x = torch.randn(T, 300, generator=torch.Generator().manual_seed(T))
    q, s = rand_weight(48, 300)
    for lo, hi in ((2.0 ** -124, 2.0 ** 100), (2.0 ** 90, 2.0 ** -60), (2.0 ** -133, 2.0 ** 120)):
        xs = (x * lo).to(torch.bfloat16)
        want, bound = ref_fp8.product(ref_fp8.rows(xs), (q, s * hi), grouped(T))
        within(fp8.linear(xs.to(device), fp8.Weight.from_quantized(q.to(device), (s * hi).to(device))), want, bound, torch.bfloat16)


@pytest.mark.parametrize("T", [1, 18])
def test_linear_large_weight(path, device, T):
    K, N = 2048, 5632
    g = torch.Generator(device=device).manual_seed(3)
    q = (torch.randn(N, K, generator=g, device=device) * 60).to(fp8.E4M3)
    s = torch.rand(44, 16, generator=g, device=device) * 1e-3 + 1e-4
    x = rand_rows(T, K, torch.bfloat16)
    want, bound = ref_fp8.product(ref_fp8.rows(x), (q.cpu(), s.cpu()), grouped(T))
    within(fp8.linear(x.to(device), fp8.Weight.from_quantized(q, s)), want, bound, torch.bfloat16)


def test_linear_nan_stays_in_its_row(path, device):
    q, s = rand_weight(64, 256)
    w = fp8.Weight.from_quantized(q.to(device), s.to(device))
    for T in (4, 200):
        x = rand_rows(T, 256, torch.bfloat16)
        clean = fp8.linear(x.to(device), w)
        x[1, 7], x[T - 1, 200] = math.nan, math.inf
        y = fp8.linear(x.to(device), w)
        assert bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[T - 1]).all())
        rest = [t for t in range(T) if t not in (1, T - 1)]
        assert torch.equal(y[rest], clean[rest])


def test_linear_row_does_not_depend_on_its_neighbours(path, device):
    """Within one size class of calls a row's bits do not depend on the other rows."""
    q, s = rand_weight(160, 640)
    w = fp8.Weight.from_quantized(q.to(device), s.to(device))
    x = rand_rows(500, 640, torch.bfloat16).to(device)
    y = fp8.linear(x, w)
    assert torch.equal(fp8.linear(x.flip(0).contiguous(), w), y.flip(0))


def test_linear_writes_only_its_output(path, device):
    q, s = rand_weight(33, 200)
    w = fp8.Weight.from_quantized(q.to(device), s.to(device))
    for T in (1, 5, 140):
        buf = torch.full((T * 33 + 64,), 7.0, device=device, dtype=torch.float16)
        x = rand_rows(T, 200, torch.float16).to(device)
        out = buf[32:32 + T * 33].view(T, 33)
        fp8.linear(x, w, out=out)
        assert torch.equal(out, fp8.linear(x, w))
        assert bool((buf[:32] == 7).all()) and bool((buf[32 + T * 33:] == 7).all())


# --------------------------------------------------------------------------------------- experts
def make_case(T, H, E, I, K, Is, gate, dtype, seed=0, pow2=False, topi=None):
    g = torch.Generator().manual_seed(seed + T)
    x = torch.randn(T, H, generator=g).to(dtype)

    def w(n, k, i):
        g2 = torch.Generator().manual_seed(seed + 7919 * i + n + 3 * k)
        q = (torch.randn(n, k, generator=g2) * 60).clamp(-448, 448).to(fp8.E4M3)
        s = torch.exp(0.5 * torch.randn(fp8.blocks(n), fp8.blocks(k), generator=g2)) / (60 * math.sqrt(k))
        return q, torch.exp2(torch.round(torch.log2(s))) if pow2 else s

    ex = [(w(I, H, 3 * e), w(I, H, 3 * e + 1), w(H, I, 3 * e + 2)) for e in range(E)]
    sh = (w(Is, H, 9001), w(Is, H, 9002), w(H, Is, 9003)) if Is else None
    if topi is None:
        topi = torch.rand(T, E, generator=g).topk(K, dim=-1).indices
    topv = torch.rand(T, K, generator=g).to(dtype)
    sg = torch.randn(T, generator=g).to(dtype) if gate else None
    return dict(x=x, ex=ex, sh=sh, topi=topi, topv=topv, sg=sg, E=E)


def on_gpu(c, device):
    def dev(t):
        return None if t is None else t.to(device)

    slab = fp8.ExpertSlab.from_quantized([tuple((dev(q), dev(s)) for q, s in t) for t in c["ex"]])
    sh = tuple(fp8.Weight.from_quantized(dev(q), dev(s)) for q, s in c["sh"]) if c["sh"] else None
    topi = dev(c["topi"])
    return dict(slab=slab, x=dev(c["x"]), topv=dev(c["topv"]), topi=topi, perm=ops.permute_build(topi, c["E"]), sh=sh, sg=dev(c["sg"]))


def oracle(c, path):
    return ref_fp8.experts(c["x"], c["topi"], c["topv"], c["ex"], c["sh"], c["sg"], grouped_gate_up(len(c["x"]), path), grouped(len(c["x"])))


CASES = [  # T, H, E, I, K, Is, gate
    (1, 64, 4, 64, 1, 0, False), (1, 256, 8, 192, 4, 320, True), (2, 192, 4, 128, 4, 128, False),
    (8, 256, 60, 128, 4, 384, True), (16, 128, 3, 320, 2, 64, True), (17, 320, 5, 64, 3, 192, False),
    (32, 256, 8, 256, 2, 448, True), (33, 128, 6, 192, 2, 128, True), (100, 192, 16, 128, 6, 0, False),
    (130, 256, 2, 64, 2, 256, False), (150, 128, 1, 128, 1, 128, True),
]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("case", CASES)
def test_experts(path, device, dtype, case):
    for pow2 in (False, True):
        c = make_case(*case, dtype, pow2=pow2)
        d = on_gpu(c, device)
        parts, shared = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], shared=d["sh"], shared_gate=d["sg"])
        want, bound, wsh, bsh = oracle(c, path)
        within(parts, want, bound, dtype)
        if c["sh"]:
            within(shared, wsh, bsh, dtype)
        else:
            assert shared is None


@pytest.mark.parametrize("T", [3, 40])
def test_every_token_on_the_same_experts(path, device, T):
    """Segments as long as the call beside empty ones.  (The ids of one token are distinct: the permutation
    build keeps one bit per token and expert.)"""
    for topi in (torch.zeros(T, 1, dtype=torch.int64) + 2, torch.tensor([[5, 1, 4]]).repeat(T, 1)):
        c = make_case(T, 128, 6, 128, topi.shape[1], 0, False, torch.bfloat16, topi=topi)
        d = on_gpu(c, device)
        parts, _ = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"])
        want, bound, _, _ = oracle(c, path)
        within(parts, want, bound, torch.bfloat16)


@pytest.mark.parametrize("T", [5, 90])
def test_host_segments_touch_only_their_rows(path, device, T):
    c = make_case(T, 128, 8, 192, 3, 0, False, torch.bfloat16)
    d = on_gpu(c, device)
    full, _ = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"])
    off = d["perm"].seg_offsets.tolist()
    parts = torch.full_like(full, 5.0)
    for order in ([6, 1], [3]):
        fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], segs=ops.seglist_host(order), parts=parts)
    for e in range(8):
        rows = slice(off[e], off[e + 1])
        if e in (6, 1, 3):
            assert torch.equal(parts[rows], full[rows])
        else:
            assert bool((parts[rows] == 5).all())
    # other slots than the expert's own number
    slab2 = fp8.ExpertSlab(10, 8, 128, 192, device)
    slab2.data.zero_()
    slab2.data[9].copy_(d["slab"].data[6])
    parts2 = torch.zeros_like(full)
    fp8.moe_ffn(slab2, d["x"], d["topv"], d["perm"], segs=ops.seglist_host([6], [9]), parts=parts2)
    assert torch.equal(parts2[off[6]:off[7]], full[off[6]:off[7]])


@pytest.mark.parametrize("T", [4, 70])
def test_shared_expert_alone(path, device, T):
    c = make_case(T, 192, 4, 64, 2, 320, True, torch.float16)
    d = on_gpu(c, device)
    _, both = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], shared=d["sh"], shared_gate=d["sg"])
    _, alone = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], shared=d["sh"], shared_gate=d["sg"], segs=ops.seglist_host([]))
    assert torch.equal(both, alone)


@pytest.mark.parametrize("T", [1, 6, 50])
def test_experts_in_a_graph_and_on_another_stream(path, device, T):
    c = make_case(T, 256, 8, 128, 2, 192, True, torch.bfloat16)
    d = on_gpu(c, device)

    def call():
        return fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], shared=d["sh"], shared_gate=d["sg"])

    want = [t.clone() for t in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):                       # two graphs at once: each has its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for i in range(3):
        d["x"].copy_(torch.randn(T, 256, generator=torch.Generator().manual_seed(i)))
        for g, _ in graphs:
            g.replay()
        eager = call()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_the_operators_together(path, device):
    """Gate, permutation, experts and combine as a layer runs them, against the same chain in 64 bits."""
    for T in (1, 9, 120):
        c = make_case(T, 256, 16, 192, 4, 256, True, torch.bfloat16, seed=11)
        d = on_gpu(c, device)
        g = torch.Generator().manual_seed(T)
        logits, bias = torch.randn(T, 16, generator=g), torch.randn(16, generator=g) * 0.1
        kw = dict(score="sigmoid", n_group=4, topk_group=2, group_score="top2", renorm=True, scale=2.5)
        topv, topi = ops.gate_select(logits.to(device), 4, bias=bias.to(device), out_dtype=torch.bfloat16, **kw)
        perm = ops.permute_build(topi, 16)
        parts, shared = fp8.moe_ffn(d["slab"], d["x"], topv, perm, shared=d["sh"], shared_gate=d["sg"])
        out = torch.empty(T, 256, device=device, dtype=torch.bfloat16)
        ops.combine(parts, perm, shared, T, 4, out)
        _, ref_i = ref_fp8.gate_select(logits, 4, bias=bias, **kw)
        assert torch.equal(topi.cpu(), ref_i)
        c["topi"], c["topv"] = ref_i, topv.cpu()
        want, bound, wsh, bsh = oracle(c, path)
        inv = perm.inv_perm.cpu().long().view(T, 4)
        total, slack = wsh.clone(), bsh + ref_fp8.half_step(torch.bfloat16, wsh.abs() + bsh)
        mag = wsh.abs() + slack
        for k in range(4):
            total += want[inv[:, k]]
            slack += bound[inv[:, k]] + ref_fp8.half_step(torch.bfloat16, want[inv[:, k]].abs() + bound[inv[:, k]])
            mag += want[inv[:, k]].abs() + bound[inv[:, k]]
        slack += 5 * 2.0 ** -8 * mag * 1.02          # combine: five additions, each rounded to bf16, of sums up to mag
        assert bool(((out.cpu().double() - total).abs() <= slack).all())


def test_no_tokens(device):
    q, s = rand_weight(32, 64)
    w = fp8.Weight.from_quantized(q.to(device), s.to(device))
    x = torch.empty(0, 64, device=device, dtype=torch.bfloat16)
    assert fp8.linear(x, w).shape == (0, 32)
    assert fp8.quantize(x).values.shape == (0, 64)


@pytest.mark.parametrize("T", [1, 33])
def test_linear_long_rows(path, device, T):
    """The longest rows: a scale for each of 512 runs."""
    K, N = 65536, 16
    q, s = rand_weight(N, K)
    x = rand_rows(T, K, torch.bfloat16)
    want, bound = ref_fp8.product(ref_fp8.rows(x), (q, s), grouped(T))
    within(fp8.linear(x.to(device), fp8.Weight.from_quantized(q.to(device), s.to(device))), want, bound, torch.bfloat16)


@pytest.mark.parametrize("T", [1, 5, 150])
def test_linear_of_many_columns(path, device, T):
    """More than 2^16 columns, as an output projection has, and not a multiple of 16."""
    K, N = 72, (1 << 16) + 43
    q, s = rand_weight(N, K)
    x = rand_rows(T, K, torch.bfloat16)
    got = fp8.linear(x.to(device), fp8.Weight.from_quantized(q.to(device), s.to(device)))
    for a, b in ((0, 128), ((1 << 16) - 128, N)):          # the first block, the last before the border and those behind
        want, bound = ref_fp8.product(ref_fp8.rows(x), (q[a:b], s[a // 128:-(-b // 128)]), grouped(T))
        within(got[:, a:b], want, bound, torch.bfloat16)


def test_linear_of_many_rows(device):
    """More rows than the streaming kernel's grid reaches, of a product small enough to be given to it."""
    T, K, N = (1 << 21) + 5, 2, 3
    q, s = rand_weight(N, K)
    x = rand_rows(64, K, torch.bfloat16)
    w = fp8.Weight.from_quantized(q.to(device), s.to(device))
    big = x.to(device).repeat(-(-T // 64), 1)[:T].contiguous()
    got = fp8.linear(big, w)
    want, bound = ref_fp8.product(ref_fp8.rows(x), (q, s), True)
    for at in (0, 1 << 20, (T - 64) // 64 * 64):
        within(got[at:at + 64], want, bound, torch.bfloat16)
    assert torch.equal(got, got[:64].repeat(-(-T // 64), 1)[:T])


def test_slots_outside_the_slab_are_refused(device):
    c = make_case(4, 128, 4, 64, 2, 0, False, torch.bfloat16, seed=3)
    d = on_gpu(c, device)
    perm = ops.permute_build(c["topi"].to(device), 4)
    few = fp8.ExpertSlab(2, 4, 128, 64, device)
    topv = c["topv"].to(device)
    with pytest.raises(ValueError, match="a slot for each"):
        fp8.moe_ffn(few, d["x"], topv, perm)
    for slot in (2, -1):
        with pytest.raises(ValueError, match="slots outside"):
            fp8.moe_ffn(few, d["x"], topv, perm, segs=ops.seglist_host([1, 3], [0, slot]))


@pytest.mark.parametrize("K", [2560, 2561, 5632])
@pytest.mark.parametrize("T", [1, 2, 9, 16, 17])
def test_linear_on_both_sides_of_the_long_rows(device, T, K):
    """20, 21 and 44 blocks: a few rows take more wavefronts from the second on; given as 16-bit rows and as 8-bit ones."""
    N = 83
    q, s = rand_weight(N, K)
    x = rand_rows(T, K, torch.bfloat16)
    w = fp8.Weight.from_quantized(q.to(device), s.to(device))
    want, bound = ref_fp8.product(ref_fp8.rows(x), (q, s), grouped(T))
    got = fp8.linear(x.to(device), w)
    within(got, want, bound, torch.bfloat16)
    assert torch.equal(fp8.linear(fp8.quantize(x.to(device)), w), got)


def test_shared_tiles_higher_than_routed_ones(device):
    """So many routed tiles that the shared expert's gate/up takes tiles of 64 rows beside routed ones of 32."""
    c = make_case(120, 64, 60, 1408, 4, 640, True, torch.bfloat16, seed=21)
    d = on_gpu(c, device)
    old = _lib.load().sparse_hip_fp8_path(2)
    try:
        parts, shared = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], shared=d["sh"], shared_gate=d["sg"])
    finally:
        _lib.load().sparse_hip_fp8_path(old)
    want, bound, wsh, bsh = oracle(c, "tiles")
    within(parts, want, bound, torch.bfloat16)
    within(shared, wsh, bsh, torch.bfloat16)


def test_linear_long_rows_in_high_tiles(device):
    """The longest rows again, in tiles of 128 rows: their scales take most of what LDS the slabs leave."""
    T, K, N = 2048, 65536, 4352
    q, s = rand_weight(256, K)
    x = rand_rows(16, K, torch.bfloat16)
    w = fp8.Weight.from_quantized(q.to(device).repeat(N // 256, 1), s.to(device).repeat(N // 256, 1))
    got = fp8.linear(x.to(device).repeat(T // 16, 1), w).view(T // 16, 16, N // 256, 256)
    assert torch.equal(got, got[:1, :, :1].expand_as(got))
    want, bound = ref_fp8.product(ref_fp8.rows(x), (q[:16], s[:1]), True)
    within(got[0, :, 0, :16], want, bound, torch.bfloat16)


def test_experts_without_tokens(device):
    c = make_case(4, 128, 4, 64, 2, 64, False, torch.bfloat16, seed=5)
    d = on_gpu(c, device)
    perm = ops.Permutation(0, 2, 4, device)          # (permute_build itself takes one token and more)
    parts, shared = fp8.moe_ffn(d["slab"], d["x"][:0], d["topv"][:0], perm, shared=d["sh"])
    assert parts.shape == (0, 128) and shared.shape == (0, 128)


def test_arguments_that_are_refused(device):
    q, s = rand_weight(32, 64)
    w = fp8.Weight.from_quantized(q.to(device), s.to(device))
    x = rand_rows(4, 64, torch.bfloat16).to(device)
    for bad in (x.t().contiguous().t(), x.float(), x[:, :32].contiguous(), x.cpu(), x[0]):
        with pytest.raises(ValueError):
            fp8.linear(bad, w)
    for out in (torch.empty(4, 32, device=device), torch.empty(4, 33, device=device, dtype=x.dtype)):
        with pytest.raises(ValueError):
            fp8.linear(x, w, out)
    with pytest.raises(ValueError):
        fp8.quantize(x.t())


@pytest.mark.parametrize("T", [4, 70])
def test_replaced_expert_keeps_its_scales(path, device, T):
    """An expert of arbitrary scales packed over one whose scales were powers of two."""
    c = make_case(T, 192, 4, 128, 2, 0, False, torch.bfloat16, seed=31, pow2=True)
    d = on_gpu(c, device)
    new = make_case(T, 192, 4, 128, 2, 0, False, torch.bfloat16, seed=77)["ex"][2]
    fp8.pack_expert_into(d["slab"].data[1], tuple((q.to(device), s.to(device)) for q, s in new), 192, 128)
    c["ex"][1] = new
    parts, _ = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"])
    want, bound, _, _ = oracle(c, path)
    within(parts, want, bound, torch.bfloat16)
    assert not d["slab"].pow2


@pytest.mark.parametrize("T", [4, 70])
def test_weight_with_changed_scales(path, device, T):
    """Scales that are written over after the weight was made count as they are now."""
    x, (q, s) = rand_rows(T, 300, torch.bfloat16), rand_weight(200, 300, pow2=True)
    w = fp8.Weight.from_quantized(q.to(device), s.to(device))
    s = s * (torch.rand(s.shape, generator=torch.Generator().manual_seed(2)) + 0.25)
    w.scales.copy_(s)
    want, bound = ref_fp8.product(ref_fp8.rows(x), (q, s), grouped(T))
    within(fp8.linear(x.to(device), w), want, bound, torch.bfloat16)
    assert not w.pow2


@pytest.mark.parametrize("T", [6, 70, 400])
def test_routed_rows_do_not_depend_on_what_else_is_in_the_call(path, device, T):
    """Experts with power-of-two scales beside others and beside a shared expert without, all in one call or each apart."""
    case = (T, 1024, 4, 704, 2, 320, True, torch.float16)
    c, odd = make_case(*case, seed=41, pow2=True), make_case(*case, seed=41)
    c["sh"], c["ex"][3] = odd["sh"], odd["ex"][3]
    c["x"] = (c["x"] * torch.exp(3 * torch.randn(1024, generator=torch.Generator().manual_seed(3))).clamp(max=200)).half()
    d = on_gpu(c, device)
    parts, shared = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], shared=d["sh"], shared_gate=d["sg"])
    apart = torch.empty_like(parts)
    for e in range(4):
        fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], segs=ops.seglist_host([e]), parts=apart)
    assert torch.equal(apart, parts)
    pure = dict(c, ex=[t if i < 3 else c["ex"][0] for i, t in enumerate(c["ex"])], sh=None)
    alone, _ = fp8.moe_ffn(on_gpu(pure, device)["slab"], d["x"], d["topv"], d["perm"])
    end = int(d["perm"].seg_offsets[3])
    assert torch.equal(alone[:end], parts[:end])


@pytest.mark.parametrize("T", [1, 2, 5])
def test_linear_into_its_own_rows_is_refused(device, T):
    """Workgroups read all of a row while others already write theirs."""
    q, s = rand_weight(256, 256)
    w = fp8.Weight.from_quantized(q.to(device), s.to(device))
    buf = torch.zeros(2 * T, 256, dtype=torch.bfloat16, device=device)
    buf[:T] = rand_rows(T, 256, torch.bfloat16).to(device)
    for out in (buf[:T], buf.view(-1)[128:128 + T * 256].view(T, 256), buf.view(-1)[T * 256 - 1:2 * T * 256 - 1].view(T, 256)):
        with pytest.raises(ValueError, match="overlaps"):
            fp8.linear(buf[:T], w, out)
    assert torch.equal(fp8.linear(buf[:T], w, buf[T:]), fp8.linear(buf[:T].clone(), w))


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("T", [1, 7, 40])
def test_experts_far_from_one(path, device, T, pow2):
    """Rows near both ends of the range beside weights whose scales bring gate and up back: runs of the lowest scale,
    scales that bf16 takes in and scales that it does not."""
    for lo, hi in ((2.0 ** -124, 2.0 ** 116), (2.0 ** -110, 2.0 ** 108), (2.0 ** 96, 2.0 ** -99), (2.0 ** 60, 2.0 ** -62)):
        c = make_case(T, 192, 3, 128, 2, 192, False, torch.bfloat16, seed=61, pow2=pow2)
        c["x"] = (c["x"].float() * lo).to(torch.bfloat16)

        def far(t):
            return (t[0][0], t[0][1] * hi), (t[1][0], t[1][1] * hi), t[2]

        c["ex"], c["sh"] = [far(t) for t in c["ex"]], far(c["sh"])
        d = on_gpu(c, device)
        parts, shared = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], shared=d["sh"])
        want, bound, wsh, bsh = oracle(c, path)
        within(parts, want, bound, torch.bfloat16)
        within(shared, wsh, bsh, torch.bfloat16)


@pytest.mark.parametrize("T", [2, 6, 150])
def test_experts_nan_stays_in_its_row(path, device, T):
    c = make_case(T, 256, 4, 192, 2, 128, True, torch.bfloat16, seed=71)
    d = on_gpu(c, device)
    clean, clean_sh = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], shared=d["sh"], shared_gate=d["sg"])
    x = d["x"].clone()
    x[0, 7], x[T - 1, 200] = math.nan, math.inf
    parts, shared = fp8.moe_ffn(d["slab"], x, d["topv"], d["perm"], shared=d["sh"], shared_gate=d["sg"])
    token = d["perm"].perm.long() // 2
    hit = (token == 0) | (token == T - 1)
    assert bool(torch.isnan(parts[hit]).all()) and torch.equal(parts[~hit], clean[~hit])
    rest = [t for t in range(T) if t not in (0, T - 1)]
    assert bool(torch.isnan(shared[0]).all()) and bool(torch.isnan(shared[T - 1]).all()) and torch.equal(shared[rest], clean_sh[rest])


def test_scales_multiplied_in_fp32_on_request(device):
    """The C entry's switch: scales that are powers of two multiplied like any others."""
    T, K, N = 300, 384, 256
    x, (q, s) = rand_rows(T, K, torch.bfloat16), rand_weight(N, K, pow2=True)
    w = fp8.Weight.from_quantized(q.to(device), s.to(device))
    rows = fp8.quantize(x.to(device))
    want, bound = ref_fp8.product(ref_fp8.rows(x), (q, s), True)
    for flag in (0, 1):
        out = torch.empty(T, N, dtype=torch.bfloat16, device=device)
        rc = ops.call_on(0, _lib.load().sparse_hip_fp8_linear, None, rows.data.data_ptr(), rows.scales.data_ptr(), 1, T, w.ref, flag,
                         out.data_ptr(), None)
        assert rc == 0
        within(out, want, bound, torch.bfloat16)
