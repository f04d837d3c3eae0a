"""Layouts, weight quantisation and refusals of the 8-bit operators and the biased selection, without a GPU.
The C entries check their arguments before any launch, so a refused call needs no device."""
import ctypes as C

import pytest
import torch

from oracle import ref_fp8
from sparse_amd import _lib, fp8, ops


def test_tiled_order_and_its_inverse():
    q = torch.randn(50, 300).to(fp8.E4M3)
    flat = fp8.tile_values(q)
    Kp = fp8.padded(300)
    assert flat.numel() == 64 * Kp
    b = q.view(torch.uint8)
    for row, k in ((0, 0), (15, 127), (16, 128), (49, 299), (33, 145), (7, 31), (7, 32)):
        at = (row // 16) * 16 * Kp + (k // 128) * 2048 + ((k // 16) % 2) * 1024 + ((k // 32) % 4) * 256 + (row % 16) * 16 + k % 16
        assert int(flat[at]) == int(b[row, k])
    assert torch.equal(fp8.untile_values(flat, 50, 300).view(torch.uint8), b)
    assert int(flat.bool().sum()) == int(b.bool().sum()), "padding is zero"


def test_weight_round_trip():
    w = torch.randn(130, 257) * 0.02
    q, s = fp8.quantize_weight(w)
    assert s.shape == (2, 3) and q.dtype == fp8.E4M3
    W = fp8.Weight.from_quantized(q, s)
    back = W.dequantize(torch.float64)
    assert torch.equal(back, ref_fp8.weight(q, s))
    # half a step of e4m3 (2^-4 of the value), or of its subnormals (2^-10 of the scale)
    step = s.repeat_interleave(128, 0)[:130].repeat_interleave(128, 1)[:, :257].double()
    assert bool(((back - w.double()).abs() <= torch.maximum(w.double().abs() * 2.0 ** -4, step * 2.0 ** -10)).all())
    with pytest.raises(ValueError, match="finite"):
        fp8.quantize_weight(torch.tensor([[1.0, float("nan")]]))


def test_power_of_two_scales_are_recognised():
    q, s = fp8.quantize_weight(torch.randn(130, 257))
    assert fp8.Weight.from_quantized(q, s).pow2
    for bad in (3.0, 0.0, -2.0, float("inf"), float("nan"), 2.0 ** -127):
        t = s.clone()
        t[1, 2] = bad
        assert not fp8.Weight.from_quantized(q, t).pow2
    ex = tuple(fp8.quantize_weight(torch.randn(*sh)) for sh in ((64, 192), (64, 192), (192, 64)))
    assert fp8.ExpertSlab.from_quantized([ex, ex]).pow2
    odd = (ex[0], (ex[1][0], ex[1][1] * 1.5), ex[2])
    assert not fp8.ExpertSlab.from_quantized([ex, odd, ex]).pow2


def test_slot_layout():
    H, I = 192, 64
    assert fp8.slot_bytes(H, I) == (2 * 64 * 256 + 192 * 128 + 4 * (2 + 2 + 2) + 255) // 256 * 256
    ex = [tuple(fp8.quantize_weight(torch.randn(*sh) * 0.02) for sh in ((I, H), (I, H), (H, I))) for _ in range(2)]
    slab = fp8.ExpertSlab.from_quantized(ex)
    at = 0
    for (q, _), (n, k) in zip(ex[1], ((I, H), (I, H), (H, I))):
        size = n * fp8.padded(k)
        assert torch.equal(fp8.untile_values(slab.data[1, at:at + size], n, k).view(torch.uint8), q.view(torch.uint8))
        at += size
    for _, s in ex[1]:
        assert torch.equal(slab.data[1, at:at + 4 * s.numel()].view(torch.float32).view(s.shape), s)
        at += 4 * s.numel()
    with pytest.raises(ValueError, match="multiples of 64"):
        fp8.ExpertSlab(1, 1, 100, 64, "cpu")
    with pytest.raises(ValueError, match="up must be"):
        fp8.ExpertSlab.from_quantized([(ex[0][0], ex[0][2], ex[0][2])])


def test_wrong_checkpoint_tensors_are_refused():
    q, s = fp8.quantize_weight(torch.randn(130, 257))
    for bad_q, bad_s in ((q.float(), s), (q, s[:1]), (q, s.double()), (q[0], s)):
        with pytest.raises(ValueError):
            fp8.Weight.from_quantized(bad_q, bad_s)


def test_python_refusals():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    w = fp8.Weight.quantize(torch.randn(32, 64))
    with pytest.raises(ValueError, match="device tensor"):
        fp8.quantize(x)
    with pytest.raises(ValueError, match="device tensor"):
        fp8.linear(x, w)
    with pytest.raises(ValueError, match="device tensor"):
        ops.gate_select(torch.zeros(2, 8), 2)


def refused(rc, *words):
    assert rc == -1
    text = _lib.last_error()
    assert all(w in text for w in words), text


def test_gate_select_refusals():
    f = _lib.load().sparse_hip_gate_select
    P = 4096   # never dereferenced: the checks come first

    def call(ldt=0, T=4, E=64, K=4, score=0, n_group=1, topk_group=1, group_score=0, odt=0, logits=P, topv=P, topi=P):
        return f(logits, ldt, None, T, E, K, score, n_group, topk_group, group_score, 0, 1.0, odt, topv, topi, None)

    refused(call(ldt=7), "dtype")
    refused(call(odt=-1), "dtype")
    refused(call(E=257), "E=257")
    refused(call(E=0), "E=0")
    refused(call(K=17), "K=17")
    refused(call(K=0), "K=0")
    refused(call(E=3, K=4), "K=4")
    refused(call(score=2), "score")
    refused(call(group_score=2), "group score")
    refused(call(n_group=5), "n_group=5")
    refused(call(E=128, n_group=128), "n_group=128")
    refused(call(n_group=4, topk_group=5), "topk_group=5")
    refused(call(n_group=4, topk_group=0), "topk_group=0")
    refused(call(n_group=32, topk_group=1, K=3), "K=3")
    refused(call(T=-1), "T=-1")
    refused(call(logits=None), "NULL")
    refused(call(topi=None), "NULL")
    assert call(T=0) == 0


def test_quantize_and_linear_refusals():
    lib = _lib.load()
    P = 4096
    refused(lib.sparse_hip_fp8_quantize(P, 9, 1, 1, P, P, None), "dtype")
    refused(lib.sparse_hip_fp8_quantize(P, 1, -1, 1, P, P, None), "T=-1")
    refused(lib.sparse_hip_fp8_quantize(P, 1, 1, 0, P, P, None), "K=0")
    refused(lib.sparse_hip_fp8_quantize(None, 1, 1, 1, P, P, None), "NULL")
    refused(lib.sparse_hip_fp8_quantize(P, 1, 1, 1, P + 4, P, None), "aligned")
    assert lib.sparse_hip_fp8_quantize(None, 1, 0, 1, None, None, None) == 0

    def lin(m=_lib.Fp8Matrix(P, P, 32, 64), x=P, xq=None, xs=None, dt=1, T=2, out=P, ws=P):
        return lib.sparse_hip_fp8_linear(x, xq, xs, dt, T, None if m is None else C.byref(m), 0, out, ws, None)

    refused(lin(dt=5), "dtype")
    refused(lin(dt=0), "bf16 or fp16")
    refused(lin(m=None), "NULL weight")
    refused(lin(m=_lib.Fp8Matrix(P, P, 0, 64)), "[0,64]")
    refused(lin(m=_lib.Fp8Matrix(P, P, 32, 1 << 21)), "must be in")
    refused(lin(m=_lib.Fp8Matrix(None, P, 32, 64)), "NULL")
    refused(lin(m=_lib.Fp8Matrix(P + 8, P, 32, 64)), "aligned")
    refused(lin(T=-3), "T=-3")
    refused(lin(x=None), "give x or")
    refused(lin(xq=P, xs=P), "give x or")
    refused(lin(out=None), "NULL output")
    refused(lin(T=3, ws=None), "workspace")
    refused(lin(T=3, ws=P + 4), "workspace")
    refused(lin(x=None, xq=P), "scales")
    assert lin(T=0) == 0


def test_moe_ffn_refusals():
    lib = _lib.load()
    P = 4096
    H, I, Is = 128, 64, 192
    stride = fp8.slot_bytes(H, I)
    mats = [_lib.Fp8Matrix(P, P, *s) for s in ((Is, H), (Is, H), (H, Is))]

    def segs(n=2, dev=False, eid=0, slot=0):
        s = _lib.SegList()
        s.n = n
        s.eids_dev = P if dev else None
        s.count_dev = None
        if n > 0:
            s.eids[0], s.slots[0] = eid, slot
        if n == 2:
            s.eids[1], s.slots[1] = 1 - eid, 1
        return s

    def call(E=4, h=H, i=I, dt=1, stride=stride, slab=P, sg=None, T=3, K=2, x=P, topv=P, parts=P, m=(None,) * 3, sh=None, ws=P):
        ex = _lib.Experts(slab, stride, None, E, h, i, dt)
        sg = segs() if sg is None else sg
        return lib.sparse_hip_fp8_moe_ffn(C.byref(ex), x, topv, P, P, C.byref(sg), T, K, parts,
                                          *(None if v is None else C.byref(v) for v in m), None, 0, sh, ws, None)

    refused(call(dt=0), "bf16 or fp16")
    refused(call(E=257), "E=257")
    refused(call(h=100), "H=100")
    refused(call(i=32), "I=32")
    refused(call(T=0), "T=0")
    refused(call(K=17), "K=17")
    refused(call(T=1 << 30, K=4), "too many rows")
    refused(call(stride=stride - 256), "slot_stride")
    refused(call(slab=None), "slab")
    refused(call(topv=None), "NULL")
    refused(call(x=None), "NULL x")
    refused(call(parts=P + 2), "aligned")
    refused(call(sg=segs(n=257)), "segment count")
    refused(call(sg=segs(n=1, eid=4)), "expert 4")
    refused(call(sg=segs(n=1, slot=-1)), "slot -1")
    refused(call(sg=segs(dev=True)), "device segment list")
    refused(call(ws=None), "workspace")
    refused(call(m=(None, mats[1], mats[2]), sh=P), "shared")
    refused(call(m=(mats[0], mats[1], _lib.Fp8Matrix(P, P, H, 100)), sh=P), "Is=100")
    refused(call(m=(mats[0], mats[0], _lib.Fp8Matrix(P, P, 64, Is)), sh=P), "down_proj")
    refused(call(m=tuple(mats), sh=None), "shared")
    assert call(sg=segs(n=0)) == 0     # nothing to do


def test_block_refusals():
    from types import SimpleNamespace as NS

    from sparse_amd.block import DistributedSparseMoeBlock
    from sparse_amd.context import DistEnv, SparseContext
    from sparse_amd.synthetic import make_mlp_block

    shape = dict(family="deepseek_shared", hidden=64, num_experts=8, inter=64, shared_inter=64)

    def make(gate=None, dtype=torch.bfloat16, **kw):
        SparseContext.reset()
        mlp = make_mlp_block(shape, dtype=dtype)
        if gate:
            mlp.gate = NS(weight=mlp.gate.weight, **gate)
        return DistributedSparseMoeBlock(0, mlp, None, DistEnv(0, 1, 0, torch.device("cpu")), num_experts=8, top_k=2, dtype=dtype, **kw)

    with pytest.raises(ValueError, match="weight_format must be"):
        make(weight_format="int4")
    with pytest.raises(ValueError, match="activations"):
        make(dtype=torch.float32, weight_format="fp8")
    with pytest.raises(ValueError, match="e_score_correction_bias"):
        make(gate=dict(topk_method="noaux_tc"))
    with pytest.raises(ValueError, match="e_score_correction_bias"):
        make(gate=dict(topk_method="greedy", e_score_correction_bias=torch.zeros(8)))
    with pytest.raises(NotImplementedError, match="scoring_func"):
        make(gate=dict(scoring_func="tanh"))


def test_an_expert_is_listed_once():
    lib = _lib.load()
    P = 4096
    s = _lib.SegList()
    s.n = 3
    for i, e in enumerate((2, 0, 2)):
        s.eids[i], s.slots[i] = e, i
    ex = _lib.Experts(P, fp8.slot_bytes(128, 64), None, 4, 128, 64, 1)
    refused(lib.sparse_hip_fp8_moe_ffn(C.byref(ex), P, P, P, P, C.byref(s), 3, 2, P, None, None, None, None, 0, None, P, None),
            "expert 2 is listed twice")


def test_workspace_of_refused_sizes():
    f = _lib.load().sparse_hip_fp8_moe_ffn_ws_bytes
    good = dict(T=8, K=2, E=8, n=8, H=128, I=64, Is=64)
    assert f(*good.values()) > 0
    for name, v in dict(T=1 << 28, K=17, E=257, n=257, H=1 << 17, I=1 << 17, Is=1 << 17).items():
        assert f(*{**good, name: v}.values()) == 0, name
    assert f(*{**good, "T": 0}.values()) == 0


def test_linear_of_a_vocabulary_is_taken():
    """More than 2^16 output columns pass the checks (and no rows are nothing to do)."""
    lib = _lib.load()
    m = _lib.Fp8Matrix(4096, 4096, 200000, 64)
    assert lib.sparse_hip_fp8_linear(4096, None, None, 1, 0, C.byref(m), 0, None, None, None) == 0
    m = _lib.Fp8Matrix(4096, 4096, (1 << 28) + 1, 64)
    refused(lib.sparse_hip_fp8_linear(4096, None, None, 1, 1, C.byref(m), 0, 4096, None, None), "must be in")


def test_native_block_refuses_an_8_bit_shared_expert():
    from sparse_amd.block import DistributedSparseMoeBlock
    from sparse_amd.context import DistEnv, SparseContext
    from sparse_amd.synthetic import make_mlp_block

    SparseContext.reset()
    mlp = make_mlp_block(dict(family="deepseek_shared", hidden=64, num_experts=8, inter=64, shared_inter=64), dtype=torch.bfloat16)
    shared = getattr(mlp, "shared_expert", None) or mlp.shared_experts
    shared.down_proj.weight = torch.nn.Parameter(shared.down_proj.weight.detach().to(torch.float8_e4m3fn), requires_grad=False)
    with pytest.raises(ValueError, match="weight_format='fp8'"):
        DistributedSparseMoeBlock(0, mlp, None, DistEnv(0, 1, 0, torch.device("cpu")), num_experts=8, top_k=2, dtype=torch.bfloat16)


@pytest.mark.parametrize("expert,matrix", [(0, "gate_proj"), (3, "up_proj"), (7, "down_proj")])
def test_native_block_refuses_one_8_bit_expert_among_others(expert, matrix):
    """8-bit values without their scales would be taken for the weights themselves."""
    from sparse_amd.block import DistributedSparseMoeBlock
    from sparse_amd.context import DistEnv, SparseContext
    from sparse_amd.synthetic import make_mlp_block

    SparseContext.reset()
    mlp = make_mlp_block(dict(family="deepseek_shared", hidden=64, num_experts=8, inter=64, shared_inter=64), dtype=torch.bfloat16)
    m = getattr(mlp.experts[expert], matrix)
    m.weight = torch.nn.Parameter(m.weight.detach().to(torch.float8_e4m3fn), requires_grad=False)
    with pytest.raises(ValueError, match="weight_format='fp8'"):
        DistributedSparseMoeBlock(0, mlp, None, DistEnv(0, 1, 0, torch.device("cpu")), num_experts=8, top_k=2, dtype=torch.bfloat16)


def test_weights_and_slabs_stay_where_their_descriptors_say():
    """The kernels go by addresses taken when a weight or slab was made: its tensors cannot be exchanged afterwards."""
    w = fp8.Weight.quantize(torch.randn(130, 257))
    assert w.desc.values_dev == w.data.data_ptr() and w.desc.scales_dev == w.scales.data_ptr()
    for name in ("data", "scales"):
        with pytest.raises(AttributeError):
            setattr(w, name, getattr(w, name).clone())
    slab = fp8.ExpertSlab(2, 2, 128, 64, "cpu")
    with pytest.raises(AttributeError):
        slab.data = slab.data.clone()


def test_weights_are_made_of_what_their_shape_needs():
    w = fp8.Weight.quantize(torch.randn(130, 257))
    fp8.Weight(w.data, w.scales, 130, 257)
    for data, scales, rows, cols in ((w.data[:-1], w.scales, 130, 257), (w.data, w.scales[:1], 130, 257),
                                     (w.data, w.scales.double(), 130, 257), (w.data.view(fp8.E4M3), w.scales, 130, 257),
                                     (w.data, w.scales, 145, 257), (w.data, w.scales, 130, 385), (w.data, w.scales.t(), 130, 257)):
        with pytest.raises(ValueError):
            fp8.Weight(data, scales, rows, cols)


def test_overlap_is_what_shares_bytes():
    t = torch.zeros(64, dtype=torch.bfloat16)
    assert fp8.overlap(t, t) and fp8.overlap(t[:32], t[31:]) and fp8.overlap(t[31:], t[:32]) and fp8.overlap(t[4:8], t)
    assert not fp8.overlap(t[:32], t[32:]) and not fp8.overlap(t[32:], t[:32]) and not fp8.overlap(t[:0], t[:0])
    assert not fp8.overlap(t, t.clone())


def test_sizes_that_32_bit_row_numbers_do_not_reach_are_refused():
    lib = _lib.load()
    P = 4096
    m = _lib.Fp8Matrix(P, P, 32, 64)
    for T in ((1 << 28) + 1, (1 << 31) - 1):
        refused(lib.sparse_hip_fp8_linear(None, P, P, 1, T, C.byref(m), 0, P, None, None), f"T={T}")
        refused(lib.sparse_hip_gate_select(P, 0, None, T, 1, 1, 0, 1, 1, 0, 0, 1.0, 0, P, P, None), f"T={T}")


def test_device_list_longer_than_the_experts_is_refused():
    """The kernels read as many entries as it says before they know how many count."""
    s = _lib.SegList()
    s.n, s.eids_dev, s.count_dev = 5, 4096, 4096
    ex = _lib.Experts(4096, fp8.slot_bytes(128, 64), None, 4, 128, 64, 1)
    refused(_lib.load().sparse_hip_fp8_moe_ffn(C.byref(ex), 4096, 4096, 4096, 4096, C.byref(s), 3, 2, 4096, None, None, None, None, 0,
                                               None, 4096, None), "4 experts")
