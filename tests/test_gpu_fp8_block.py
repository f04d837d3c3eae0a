"""The layer block with 8-bit experts and with gates balanced by a bias, resident and offloaded."""
from types import SimpleNamespace as NS

import pytest
import torch

from oracle import ref_fp8
from sparse_amd import fp8
from sparse_amd.block import DistributedSparseMoeBlock
from sparse_amd.context import DistEnv, Metrics, SparseContext
from sparse_amd.synthetic import make_hidden, make_mlp_block

pytestmark = pytest.mark.gpu
QWEN = dict(family="qwen_shared", hidden=256, num_experts=12, inter=192, top_k=4, shared_inter=320)
DEEP = dict(family="deepseek_shared", hidden=192, num_experts=16, inter=128, top_k=3, shared_inter=128)


def block(mlp, shape, device, dtype=torch.bfloat16, **kw):
    return DistributedSparseMoeBlock(0, mlp, None, DistEnv(0, 1, 0, device), num_layers=1, num_experts=shape["num_experts"],
                                     top_k=shape["top_k"], dtype=dtype, metrics=Metrics(), **kw)


def biased(mlp, shape, seed=3):
    g = torch.Generator().manual_seed(seed)
    mlp.gate = NS(weight=mlp.gate.weight, e_score_correction_bias=torch.randn(shape["num_experts"], generator=g) * 0.05,
                  n_group=4, topk_group=2, routed_scaling_factor=2.5)
    mlp.norm_topk_prob = True
    return mlp


def triple(m):
    return tuple(fp8.quantize_weight(w.weight.float()) for w in (m.gate_proj, m.up_proj, m.down_proj))


def run(blk, x, device):
    T, H = x.shape
    out = blk(x.view(T, 1, H).to(device))
    out, logits = out if isinstance(out, tuple) else (out, None)
    return out.view(T, H), logits


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [QWEN, DEEP])
@pytest.mark.parametrize("T", [1, 2, 8, 40])
def test_resident_block_against_the_oracle(device, dtype, shape, T):
    SparseContext.reset()
    mlp = make_mlp_block(shape, dtype=dtype, seed=1, std=0.05)
    blk = block(mlp, shape, device, dtype, weight_format="fp8")
    x = make_hidden(T, shape["hidden"], dtype, seed=7)
    out, _ = run(blk, x, device)
    ws = blk._workspace(T)
    sh = mlp.shared_expert if shape is QWEN else mlp.shared_experts
    want, bound, wsh, bsh = ref_fp8.experts(x, ws.topi.cpu(), ws.topv.cpu(), [triple(m) for m in mlp.experts], triple(sh),
                                            ws.shared_gate.cpu() if shape is QWEN else None, False, True)
    parts = ws.parts.cpu().double()
    assert bool(((parts - want).abs() <= bound + ref_fp8.half_step(dtype, want.abs() + bound)).all())
    shared = ws.shared_out.cpu().double()
    assert bool(((shared - wsh).abs() <= bsh + ref_fp8.half_step(dtype, wsh.abs() + bsh)).all())
    # combine: the rows in ascending expert id, each addition rounded, the shared expert last
    K, inv = shape["top_k"], ws.perm.inv_perm.cpu().long().view(T, -1)
    total = torch.zeros(T, shape["hidden"], dtype=dtype)
    for p in inv.sort(dim=1).values.t():
        total = total + ws.parts.cpu()[p]
    assert torch.equal(out.cpu(), total + ws.shared_out.cpu()) and inv.shape[1] == K


@pytest.mark.parametrize("shape", [QWEN, DEEP])
@pytest.mark.parametrize("T", [2, 8, 100])
def test_offloaded_block_gives_the_resident_bits(device, shape, T):
    SparseContext.reset()
    mlp = make_mlp_block(shape, dtype=torch.bfloat16, seed=2, std=0.05)
    a = block(mlp, shape, device, weight_format="fp8")
    b = block(mlp, shape, device, weight_format="fp8", expert_offload="cpu", expert_cache=3)
    assert b.arena.expert_bytes == fp8.slot_bytes(shape["hidden"], shape["inter"])
    for call in range(3):
        x = make_hidden(T, shape["hidden"], torch.bfloat16, seed=20 + call)
        SparseContext.begin_runtime_call(call)
        want, _ = run(a, x, device)
        got, _ = run(b, x, device)
        assert torch.equal(got, want)
    assert b.metrics.cache_miss_count > 0
    assert b.metrics.demand_h2d_bytes % b.arena.expert_bytes == 0


def test_checkpoint_modules_keep_their_own_scales(device):
    SparseContext.reset()
    mlp = make_mlp_block(DEEP, dtype=torch.bfloat16, seed=4, std=0.05)

    def eight(m):
        q, s = fp8.quantize_weight(m.weight.float())
        f = torch.rand(s.shape, generator=torch.Generator().manual_seed(s.numel())) + 0.5
        return NS(weight=q, weight_scale_inv=s * f)

    eighted = NS(gate=mlp.gate, experts=[NS(gate_proj=eight(m.gate_proj), up_proj=eight(m.up_proj), down_proj=eight(m.down_proj))
                                         for m in mlp.experts],
                 shared_experts=mlp.shared_experts)
    with pytest.raises(ValueError, match="weight_format"):
        block(eighted, DEEP, device)
    blk = block(eighted, DEEP, device, weight_format="fp8")
    assert not blk.slab.pow2
    x = make_hidden(6, DEEP["hidden"], torch.bfloat16, seed=8)
    run(blk, x, device)
    ws = blk._workspace(6)
    ex = [tuple((m.weight, m.weight_scale_inv) for m in (e.gate_proj, e.up_proj, e.down_proj)) for e in eighted.experts]
    want, bound, _, _ = ref_fp8.experts(x, ws.topi.cpu(), ws.topv.cpu(), ex, None, None, False, True)
    assert bool(((ws.parts.cpu().double() - want).abs() <= bound + ref_fp8.half_step(torch.bfloat16, want.abs() + bound)).all())
    del eighted.experts[0].gate_proj.weight_scale_inv
    with pytest.raises(ValueError, match="weight_scale_inv"):
        block(eighted, DEEP, device, weight_format="fp8")


@pytest.mark.parametrize("T", [1, 20, 70])
@pytest.mark.parametrize("weight_format", ["native", "fp8"])
def test_biased_gate(device, T, weight_format):
    SparseContext.reset()
    mlp = biased(make_mlp_block(DEEP, dtype=torch.bfloat16, seed=5, std=0.05), DEEP)
    blk = block(mlp, DEEP, device, weight_format=weight_format)
    assert blk.gate_score == "sigmoid" and blk.gate_group_score == "top2" and (blk.n_group, blk.topk_group) == (4, 2)
    x = make_hidden(T, DEEP["hidden"], torch.bfloat16, seed=9)
    topv, topi, _ = blk._routing_router(x.to(device))
    from sparse_amd import ops
    logits, _ = ops.router_logits(x.to(device), blk.gate_weight, None, torch.float32)
    want_v, want_i = ref_fp8.gate_select(logits.cpu(), 3, "sigmoid", mlp.gate.e_score_correction_bias, 4, 2, "top2", True, 2.5)
    assert torch.equal(topi.cpu(), want_i)
    tol = ref_fp8.half_step(torch.bfloat16, want_v) * (1 + 2.0 ** -8)
    assert bool(((topv.cpu().double() - want_v).abs() <= tol + want_v.abs() * 2.0 ** -24).all())
    out, _ = run(blk, x, device)
    assert bool(torch.isfinite(out).all())


def test_block_in_a_graph(device):
    SparseContext.reset()
    mlp = biased(make_mlp_block(DEEP, dtype=torch.bfloat16, seed=6, std=0.05), DEEP)
    blk = block(mlp, DEEP, device, weight_format="fp8")
    x = make_hidden(8, DEEP["hidden"], torch.bfloat16, seed=10).to(device).view(8, 1, -1)
    blk(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = blk(x)
    for i in range(4):
        x.copy_(make_hidden(8, DEEP["hidden"], torch.bfloat16, seed=30 + i).view(8, 1, -1))
        graph.replay()
        want = blk(x.clone())
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_segment_timing_of_an_8_bit_block(device, monkeypatch):
    SparseContext.reset()
    mlp = make_mlp_block(QWEN, dtype=torch.bfloat16, seed=11, std=0.05)
    blk = block(mlp, QWEN, device, weight_format="fp8")
    x = make_hidden(5, QWEN["hidden"], torch.bfloat16, seed=12)
    want, _ = run(blk, x, device)
    monkeypatch.setenv("SPARSE_EXPERT_TIMING", "1")
    got, _ = run(blk, x, device)
    assert torch.equal(got, want) and blk.metrics.moe_timing_calls == 3


def test_deepseek_v3_model_with_swapped_blocks(device):
    """A tiny model whose gate is balanced by a bias: the swapped blocks read bias, groups and scaling from its
    gate module and reproduce its logits and greedy continuation."""
    pytest.importorskip("transformers")
    try:
        from transformers import DeepseekV3Config, DeepseekV3ForCausalLM
    except ImportError:
        pytest.skip("this transformers has no DeepSeek-V3")
    from sparse_amd import harness
    cfg = DeepseekV3Config(vocab_size=160, hidden_size=128, intermediate_size=256, moe_intermediate_size=64,
                           num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=4, n_routed_experts=16,
                           num_experts_per_tok=4, n_shared_experts=1, first_k_dense_replace=1, n_group=4, topk_group=2,
                           norm_topk_prob=True, routed_scaling_factor=2.5, max_position_embeddings=128, kv_lora_rank=32,
                           q_lora_rank=None, qk_rope_head_dim=16, qk_nope_head_dim=16, v_head_dim=32)
    torch.manual_seed(1)
    model = DeepseekV3ForCausalLM(cfg).eval()
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() >= 2:
                p.mul_(3.0)
        for layer in model.model.layers[1:]:
            layer.mlp.gate.e_score_correction_bias.uniform_(0.0, 0.3)
    model = model.to(torch.float32).to(device)
    ids = torch.tensor([[5, 17, 42, 99, 3, 64], [7, 7, 120, 33, 8, 1]], device=device)
    mask = torch.ones_like(ids)
    SparseContext.reset()
    with torch.no_grad():
        want_logits = model(input_ids=ids, attention_mask=mask, use_cache=False, return_dict=True).logits.float().cpu()
        want_ids = harness.greedy_decode(model, ids, mask, 5).cpu()
    SparseContext.reset()
    blocks = harness.install_sparse_blocks(model, env=DistEnv(0, 1, 0, device), dtype=torch.float32, metrics=Metrics())
    assert blocks[0].gate_bias is not None and blocks[0].gate_score == "sigmoid"
    assert (blocks[0].n_group, blocks[0].topk_group, blocks[0].routed_scaling_factor) == (4, 2, 2.5)
    with torch.no_grad():
        harness.begin_request()
        SparseContext.current_phase = "prefill"
        SparseContext.begin_runtime_call(0)
        got_logits = model(input_ids=ids, attention_mask=mask, use_cache=False, return_dict=True).logits.float().cpu()
        torch.testing.assert_close(got_logits, want_logits, rtol=2e-4, atol=2e-4)
        harness.begin_request()
        got_ids = harness.greedy_decode(model, ids, mask, 5).cpu()
    assert torch.equal(got_ids, want_ids)


@pytest.mark.parametrize("T", [8, 120, 500])
def test_offloaded_block_gives_the_resident_bits_beside_a_shared_expert_of_other_scales(device, T):
    """Routed experts quantised at load (scales that are powers of two), a shared expert with a checkpoint's own ones:
    the routed rows are the same whether they run in the shared expert's call or in their own."""
    shape = dict(QWEN, hidden=1024, inter=704)
    SparseContext.reset()
    mlp = make_mlp_block(shape, dtype=torch.float16, seed=13, std=0.05)

    def eight(m):
        q, s = fp8.quantize_weight(m.weight.float())
        return NS(weight=q, weight_scale_inv=s * (torch.rand(s.shape, generator=torch.Generator().manual_seed(s.numel())) + 0.5))

    sh = mlp.shared_expert
    mixed = NS(gate=mlp.gate, experts=mlp.experts, shared_expert_gate=mlp.shared_expert_gate,
               shared_expert=NS(gate_proj=eight(sh.gate_proj), up_proj=eight(sh.up_proj), down_proj=eight(sh.down_proj)))
    a = block(mixed, shape, device, torch.float16, weight_format="fp8")
    b = block(mixed, shape, device, torch.float16, weight_format="fp8", expert_offload="cpu", expert_cache=3)
    assert a.slab.pow2 and not a.shared_weights[0].pow2
    for call in range(2):
        x = make_hidden(T, shape["hidden"], torch.float16, seed=50 + call)
        x = (x * torch.exp(3 * torch.randn(1024, generator=torch.Generator().manual_seed(3))).clamp(max=200)).half()
        SparseContext.begin_runtime_call(call)
        want, _ = run(a, x, device)
        got, _ = run(b, x, device)
        assert torch.equal(got, want)


def test_costs_of_an_8_bit_block_are_measured(device, monkeypatch):
    """Calibration runs the 8-bit experts and uploads the bytes of one of their slots."""
    from sparse_amd import local_policy, ops
    SparseContext.reset()
    blk = block(make_mlp_block(QWEN, dtype=torch.bfloat16, seed=14, std=0.05), QWEN, device, weight_format="fp8")
    sizes, upload = [], ops.expert_upload_async
    monkeypatch.setattr(ops, "expert_upload_async", lambda d, h, n, s, e: (sizes.append(n), upload(d, h, n, s, e))[1])
    costs = local_policy.measure_costs(blk, batches=(1, 4, 40), repeats=3)
    assert all(v >= 0 for v in costs.values()) and costs["next_attention_ms"] > 0
    assert max(sizes) == blk.slab.expert_bytes == fp8.slot_bytes(QWEN["hidden"], QWEN["inter"])
    x = make_hidden(4, QWEN["hidden"], torch.bfloat16, seed=15)
    run(blk, x, device)                       # and leaves the block as it was
