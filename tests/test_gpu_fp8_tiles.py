"""The tiles of 8-bit products of many rows: every height, full and with each number of 32-row sub-tiles at a segment's
end, several k slabs that end inside a block, scales of every kind.  The height that a case is about is read off the
size of the workspace the library asks for.

Calls consist of a few distinct tokens, each repeated many times, so that the 64-bit oracle stays small: every
repetition has to have the bits of the first, whichever tile and sub-tile it falls into."""

import pytest
import torch

from oracle import ref_fp8
from sparse_amd import _lib, fp8, ops

from .test_gpu_fp8 import make_case, on_gpu, rand_rows, rand_weight, within

pytestmark = pytest.mark.gpu
H, I, E, K = 704, 832, 6, 2


def up(n, m):
    return -(-n // m)


def queue_bytes(T, Is, rows, shared_rows):
    """Bytes of the tile queues with tiles of that many rows."""
    cols = 128 if rows == 32 else 256
    mt = up(T * K, rows) + E
    entries = 2 + mt * (up(I, 128) + up(H, cols))
    if Is:
        entries += up(T, shared_rows) * up(Is, 128) + up(T, rows) * up(H, cols)
    return up(256 + 16 * entries, 256) * 256


def heights(T, Is):
    """(rows of routed tiles, rows of the shared expert's gate/up tiles) that the library takes."""
    lib = _lib.load()
    before = lib.sparse_hip_fp8_path(2)
    total = lib.sparse_hip_fp8_moe_ffn_ws_bytes(T, K, E, E, H, I, Is)
    lib.sparse_hip_fp8_path(before)
    total -= up(2 * T * fp8.padded(H), 256) * 256                 # x in bf16
    for rows, k in ((T * K, I),) + (((T, Is),) if Is else ()):
        total -= up(rows * fp8.padded(k), 256) * 256 + up(rows * fp8.blocks(k), 256) * 256
    fits = [(r, s) for r in (32, 64, 128) for s in (32, 64, 128) if s >= r and queue_bytes(T, Is, r, s) == total]
    assert fits, total
    return fits[0] if Is else (fits[0][0], None)


# lengths of the segments beyond whole tiles of 128: remainders of 1..32, 33..64, 65..96 and 97..127 rows
ENDS = [(17, 33, 47, 63), (64, 1, 31, 96), (97, 15, 81, 32)]


def repeated(T_tiles, ends, Is, gate, dtype, pow2, seed=0):
    """Sixteen tokens, token d on experts d % 4 and d % 4 + 1 (nobody on the last one), in an order without one."""
    counts = [128 * t + e for t, e in zip(T_tiles, ends)]
    ids = []
    for a, n in enumerate(counts):
        ids += [(a + 4 * (i % 4)) for i in range(n)]
    g = torch.Generator().manual_seed(seed)
    ids = torch.tensor(ids)[torch.randperm(len(ids), generator=g)]
    topi = torch.stack([torch.arange(16) % 4, torch.arange(16) % 4 + 1], 1)
    c = make_case(16, H, E, I, K, Is, gate, dtype, seed=seed, pow2=pow2, topi=topi)
    c["x"] = (c["x"] * torch.exp(torch.randn(H, generator=g))).to(dtype)
    big = dict(c, x=c["x"][ids], topi=topi[ids], topv=c["topv"][ids], sg=c["sg"][ids] if gate else None)
    return c, big, ids, counts


def check_repeated(c, big, ids, device, oracle):
    d = on_gpu(big, device)
    parts, shared = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], shared=d["sh"], shared_gate=d["sg"])
    want, bound, wsh, bsh = oracle(c)
    # permuted rows in the order (expert, flat index), of the sixteen tokens and of their repetitions
    flat = big["topi"].reshape(-1)
    order = torch.sort(flat, stable=True).indices
    small = torch.sort(c["topi"].reshape(-1), stable=True).indices
    place = torch.empty(16 * K, dtype=torch.int64)
    place[small] = torch.arange(16 * K)
    row = place[ids[order // K] * K + order % K]                  # row of `want` that row p of `parts` repeats
    first = torch.full((16 * K,), len(row), dtype=torch.int64).scatter_reduce(0, row, torch.arange(len(row)), "amin")
    got = parts.cpu()
    assert torch.equal(got, got[first[row]]), "a row depends on its place"
    within(got[first], want, bound, got.dtype)
    if c["sh"]:
        got = shared.cpu()
        first = torch.full((16,), len(ids), dtype=torch.int64).scatter_reduce(0, ids, torch.arange(len(ids)), "amin")
        assert torch.equal(got, got[first[ids]]), "a shared row depends on its place"
        within(got[first], wsh, bsh, got.dtype)


# tiles of 128 rows in the four kinds of tokens -> heights of the routed tiles and of the shared expert's gate/up tiles
TILES = {(64, 64): (2, 2, 2, 2), (64, 128): (4, 4, 3, 3), (128, 128): (5, 5, 4, 4)}


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Is,gate", [(448, True), (320, False), (0, False)])
@pytest.mark.parametrize("ends", ENDS)
@pytest.mark.parametrize("tiles", list(TILES))
def test_experts_in_tiles_of(device, tiles, ends, Is, gate, dtype, pow2):
    c, big, ids, counts = repeated(TILES[tiles], ends, Is, gate, dtype, pow2, seed=sum(tiles))
    assert heights(len(ids), Is) == (tiles if Is else (tiles[0], None))
    lengths = [counts[0], counts[0] + counts[1], counts[1] + counts[2], counts[2] + counts[3], counts[3]]
    if ends == ENDS[0]:
        assert {up(n % tiles[0], 32) for n in lengths} == set(range(1, tiles[0] // 32 + 1))
    before = _lib.load().sparse_hip_fp8_path(2)
    try:
        check_repeated(c, big, ids, device,
                       lambda c: ref_fp8.experts(c["x"], c["topi"], c["topv"], c["ex"], c["sh"], c["sg"], True, True))
    finally:
        _lib.load().sparse_hip_fp8_path(before)


@pytest.mark.parametrize("tiles", list(TILES))
def test_experts_of_both_kinds_of_scales(device, tiles):
    """Some experts' scales are powers of two and go into the instruction, others' and the shared one's are not."""
    c, big, ids, _ = repeated(TILES[tiles], ENDS[0], 448, True, torch.float16, True, seed=9)
    odd, _, _, _ = repeated(TILES[tiles], ENDS[0], 448, True, torch.float16, False, seed=9)
    for k in ("ex", "sh"):
        both = [odd[k][i] if k == "sh" or i % 2 else c[k][i] for i in range(len(c[k]))]
        c[k] = big[k] = tuple(both)
    assert heights(len(ids), 448) == tiles
    check_repeated(c, big, ids, device,
                   lambda c: ref_fp8.experts(c["x"], c["topi"], c["topv"], c["ex"], c["sh"], c["sg"], True, True))


@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,N,rows", [(64 * 24 + 40, 2817, 64), (64 * 25 + 7, 2816, 64), (128 * 22 + 70, 2817, 128),
                                      (128 * 22 + 20, 2818, 128), (128 * 23 + 60, 2817, 128), (128 * 23 - 3, 2820, 128)])
def test_linear_in_wide_tiles(device, T, N, rows, dtype, pow2):
    """The last tile holds one to four sub-tiles; odd K and N; scales of one block that is and one that is not."""
    K = 1001
    assert [r for r in (32, 64) if T // r * up(N, 256) <= 512][:1] == ([64] if rows == 64 else [])
    x, (q, s) = rand_rows(16, K, dtype), rand_weight(N, K, pow2=pow2)
    if pow2:
        s[5, 3] *= 1.25                  # the tile of columns 512 .. 767 has one scale that is no power of two
    ids = torch.randint(0, 16, (T,), generator=torch.Generator().manual_seed(T))
    ids[-16:] = torch.arange(16)
    w = fp8.Weight.from_quantized(q.to(device), s.to(device))
    got = fp8.linear(x[ids].to(device), w).cpu()
    first = torch.full((16,), T, dtype=torch.int64).scatter_reduce(0, ids, torch.arange(T), "amin")
    assert torch.equal(got, got[first[ids]]), "a row depends on its place"
    want, bound = ref_fp8.product(ref_fp8.rows(x), (q, s), True)
    within(got[first], want, bound, dtype)
    # and against the product as it is defined, without the instruction's cut-off
    want, bound = ref_fp8.product(ref_fp8.rows(x), (q, s), False)
    within(got[first], want, bound + ref_fp8.cut_bound(ref_fp8.rows(x), (q, s)), dtype)


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("which", [1, 2])
def test_small_products_against_their_formula(device, which, T):
    """Both families of kernels at most a derived distance from the operators' own formulas."""
    c = make_case(T, 320, 4, 192, 2, 256, True, torch.float16, seed=51)
    x, w = rand_rows(T, 700, torch.float16), rand_weight(300, 700)
    d = on_gpu(c, device)
    before = _lib.load().sparse_hip_fp8_path(which)
    try:
        y = fp8.linear(x.to(device), fp8.Weight.from_quantized(*(t.to(device) for t in w)))
        parts, shared = fp8.moe_ffn(d["slab"], d["x"], d["topv"], d["perm"], shared=d["sh"], shared_gate=d["sg"])
    finally:
        _lib.load().sparse_hip_fp8_path(before)
    want, bound = ref_fp8.product(ref_fp8.rows(x), w, False)
    within(y, want, bound + ref_fp8.cut_bound(ref_fp8.rows(x), w), torch.float16)
    xq, flat = ref_fp8.rows(c["x"]), c["topi"].reshape(-1)
    at = 0
    for e in range(4):
        items = torch.nonzero(flat == e).reshape(-1)
        f = c["topv"].double().reshape(-1)[items, None]
        want, bound = ref_fp8.swiglu_formula(xq[items // 2], *c["ex"][e])
        within(parts[at:at + len(items)], want * f, bound * f, torch.float16)
        at += len(items)
    f = torch.sigmoid(c["sg"].double())[:, None]
    want, bound = ref_fp8.swiglu_formula(xq, *c["sh"])
    within(shared, want * f, bound * f + 2.0 ** -20 * (want * f).abs(), torch.float16)
