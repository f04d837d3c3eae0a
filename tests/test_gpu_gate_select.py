"""Biased expert selection through the C ABI against the 64-bit oracle: ids equal, weights within the one
rounding to their type."""
import math

import pytest
import torch

from oracle import ref_fp8
from sparse_amd import ops

pytestmark = pytest.mark.gpu


def check(logits, k, out_dtype, device, **kw):
    bias = kw.pop("bias", None)
    topv, topi = ops.gate_select(logits.to(device), k, bias=None if bias is None else bias.to(device),
                                 out_dtype=out_dtype, **kw)
    ref_v, ref_i = ref_fp8.gate_select(logits, k, bias=bias, **kw)
    assert topi.dtype == torch.int64 and torch.equal(topi.cpu(), ref_i)
    got = topv.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref_v))
    # one rounding to out_dtype, by way of fp32 for the 16-bit types; the 64-bit steps before it are good to 2^-48
    tol = ref_fp8.half_step(out_dtype, ref_v) * (1 + 2.0 ** -8) + ref_v.abs() * 2.0 ** -24 * (out_dtype != torch.float32)
    fine = ~torch.isnan(ref_v)
    assert bool(((got - ref_v).abs()[fine] <= tol[fine]).all())


GROUPS = [(1, 1), (8, 4), (4, 1), (2, 2)]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k", [(1, 8, 1), (1, 256, 8), (3, 64, 16), (5, 160, 6), (70, 256, 8), (7, 1, 1), (9, 60, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_scores_and_bias(device, score, T, E, k, dtype):
    g = torch.Generator().manual_seed(T * 1000 + E)
    logits = (torch.randn(T, E, generator=g) * 2).to(dtype)
    bias = torch.randn(E, generator=g) * 0.05
    for renorm, scale in ((False, 1.0), (True, 2.5)):
        check(logits, k, dtype, device, score=score, bias=bias, renorm=renorm, scale=scale)
        check(logits, k, torch.float32, device, score=score, renorm=renorm, scale=scale)


@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("n_group,topk_group", GROUPS)
@pytest.mark.parametrize("E", [64, 160, 256, 8])
def test_groups(device, group_score, n_group, topk_group, E):
    g = torch.Generator().manual_seed(E + n_group)
    logits = torch.randn(33, E, generator=g)
    bias = torch.randn(E, generator=g) * 0.1
    k = min(6, topk_group * (E // n_group))
    for score in ("softmax", "sigmoid"):
        check(logits, k, torch.bfloat16, device, score=score, bias=bias, n_group=n_group, topk_group=topk_group,
              group_score=group_score, renorm=True)


def test_odd_groups_and_sixty_four_of_them(device):
    g = torch.Generator().manual_seed(5)
    check(torch.randn(11, 60, generator=g), 5, torch.float32, device, score="sigmoid", n_group=12, topk_group=5, group_score="top2")
    check(torch.randn(11, 192, generator=g), 3, torch.float32, device, score="sigmoid", n_group=64, topk_group=1, group_score="top2")
    check(torch.randn(11, 64, generator=g), 7, torch.float32, device, score="softmax", n_group=64, topk_group=7, group_score="top2")


def test_ties_go_to_the_lower_id(device):
    logits = torch.zeros(4, 96)
    logits[1, 50:] = 1.0
    logits[2, ::2] = -3.0
    bias = torch.zeros(96)
    for kw in (dict(), dict(n_group=4, topk_group=2), dict(n_group=4, topk_group=2, group_score="top2")):
        for score in ("softmax", "sigmoid"):
            check(logits, 6, torch.float32, device, score=score, **kw)
            check(logits, 6, torch.float32, device, score=score, bias=bias, **kw)


def test_scores_closer_than_one_fp32_rounding(device):
    """Pairs that 32 bits cannot tell apart are ranked by their 64-bit scores."""
    E = 128
    logits = torch.linspace(-1, 1, E).repeat(16, 1)
    p = torch.sigmoid(logits[0].double())
    bias = (0.75 - p).float()            # score + bias is 0.75 up to the rounding of the bias
    check(logits, 8, torch.float32, device, score="sigmoid", bias=bias)
    check(logits, 8, torch.float32, device, score="sigmoid", bias=bias, n_group=8, topk_group=3, group_score="top2")


def test_masked_and_empty_rows(device):
    g = torch.Generator().manual_seed(6)
    logits = torch.randn(6, 40, generator=g)
    logits[0] = -math.inf
    logits[1, 3:] = -math.inf
    logits[2, ::2] = torch.finfo(torch.float32).min
    logits[3, :] = torch.finfo(torch.float32).min
    bias = torch.randn(40, generator=g) * 0.1
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            check(logits, 5, torch.float32, device, score=score, bias=b, renorm=False)
            check(logits, 5, torch.float32, device, score=score, bias=b, renorm=True, n_group=5, topk_group=2)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_ids_stay_distinct_beside_nan_and_infinity(device, bad):
    logits = torch.randn(8, 64, generator=torch.Generator().manual_seed(7))
    logits[0, 5] = bad
    logits[1] = bad
    logits[2, ::3] = bad
    bias = torch.zeros(64)
    bias[9] = math.inf
    bias[10] = -math.inf
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            for kw in (dict(), dict(n_group=8, topk_group=4, group_score="top2")):
                topv, topi = ops.gate_select(logits.to(device), 8, score=score, bias=None if b is None else b.to(device),
                                             renorm=True, **kw)
                ids = topi.cpu()
                assert int(ids.min()) >= 0 and int(ids.max()) < 64
                assert all(len(set(row.tolist())) == 8 for row in ids)
                # rows without a special value are untouched by the ones beside them
                ref_v, ref_i = ref_fp8.gate_select(logits[3:], 8, score=score, bias=b, renorm=True, **kw)
                if b is None:
                    assert torch.equal(ids[3:], ref_i)
                    assert float((topv.cpu()[3:].double() - ref_v).abs().max()) <= 2.0 ** -23


def test_a_prompt_and_a_single_token_agree(device):
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(4099, 256, generator=g).to(device)
    bias = (torch.randn(256, generator=g) * 0.1).to(device)
    kw = dict(score="sigmoid", bias=bias, n_group=8, topk_group=4, group_score="top2", renorm=True, scale=2.5)
    topv, topi = ops.gate_select(logits, 8, **kw)
    for t in (0, 1, 2047, 4098):
        v, i = ops.gate_select(logits[t:t + 1].contiguous(), 8, **kw)
        assert torch.equal(v[0], topv[t]) and torch.equal(i[0], topi[t])


def test_graph_replay_and_other_stream(device):
    logits = torch.randn(17, 64, device=device)
    topv = torch.empty(17, 6, device=device)
    topi = torch.empty(17, 6, device=device, dtype=torch.int64)
    ops.gate_select(logits, 6, score="sigmoid", topv=topv, topi=topi)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ops.gate_select(logits, 6, score="sigmoid", topv=topv, topi=topi)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        ops.gate_select(logits, 6, score="sigmoid", topv=topv, topi=topi)
    for i in range(4):
        logits.copy_(torch.randn(17, 64, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        want_v, want_i = ops.gate_select(logits.clone(), 6, score="sigmoid")
        torch.cuda.synchronize()
        assert torch.equal(topv, want_v) and torch.equal(topi, want_i)


def test_no_rows(device):
    topv, topi = ops.gate_select(torch.empty(0, 16, device=device), 4)
    assert topv.shape == (0, 4) and topi.shape == (0, 4)


def test_group_sums_that_cancel(device):
    """The two best of each group are large and of opposite sign, so that their sums differ by less than 32 bits hold of
    the terms: the 64-bit sums decide (0.80088 against 0.80067: the first group)."""
    logits = torch.tensor([[0.00351563, -0.84729785, 0.00429688, -0.84920335]])
    bias = torch.tensor([16384.0, -16384.0, 16384.0, -16384.0])
    for _ in range(2):
        check(logits, 1, torch.float32, device, score="sigmoid", bias=bias, n_group=2, topk_group=1, group_score="top2")
        logits, bias = logits.view(2, 2).flip(0).reshape(1, 4).contiguous(), bias.clone()


@pytest.mark.parametrize("size", [1.0, 16.0, 128.0, 256.0, 1024.0, 16384.0, 1e5])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_large_biases_of_both_signs(device, score, size):
    """Groups of two whose sums nearly tie beside biases of ``size`` and ``-size``."""
    g = torch.Generator().manual_seed(int(size))
    T = 3000
    base = torch.randn(T, 1, 2, generator=g)
    logits = (base + torch.randn(T, 4, 2, generator=g) * 2.0 ** -6).reshape(T, 8).contiguous()
    bias = torch.tensor([size, -size]).repeat(4)
    for topk_group in (1, 2):
        check(logits, 1, torch.float32, device, score=score, bias=bias, n_group=4, topk_group=topk_group, group_score="top2")
    check(logits, 2, torch.float32, device, score=score, bias=bias, n_group=4, topk_group=3, group_score="max")
