"""``DistributedSparseMoeBlock``: the MoE layer of louislichen/SPARSE on one MI355X.

Keeps the reference block's constructor keywords, ``forward(hidden[B,S,H])`` signature,
return convention and lifecycle hooks (utils/eval_core.py:4408-4440, :16418-16563,
:6097-6147, :16565-16659) and runs the layer through the HIP kernels behind the C ABI:

    router_logits -> gate_topk -> permute_build -> shared_expert
                  -> grouped_swiglu (resident: one device-ordered launch pair;
                     offloaded: batches ordered by the residency policy)
                  -> combine

``expert_offload="gpu"`` keeps every expert in an HBM slab and never touches the host
during ``forward`` (capturable in a HIP graph).  ``expert_offload="cpu"`` keeps experts in
pinned host memory and a per-layer HBM cache of ``expert_cache`` slots; ``forward`` then
synchronises once per call to learn which experts were routed, exactly where the
reference's ``torch.where`` / ``.tolist()`` calls synchronise.
"""
from __future__ import annotations

import os
from typing import Any, Dict, List, Optional, Sequence, Tuple

import torch
import torch.nn.functional as F
from torch import nn

from . import fp8, ops
from ._lru import LruTable
from .context import DistEnv, Metrics, SparseContext
from .residency import Backend, LayerResidency, ResidencyConfig
from .rs import fused_scout, router_topk_feature, stable_topk, topk_for_planning
from .weights import ExpertSlab, HostExpertArena, tile_weight


def _is_silu(fn: Any) -> bool:
    if fn is None or fn is F.silu or isinstance(fn, nn.SiLU) or getattr(fn, "__name__", "") == "silu":
        return True
    # Hugging Face wraps it in its own module class in some versions
    return type(fn).__name__.lower() in ("silu", "siluactivation")


def _bump(metrics: Any, name: str, value: int) -> None:
    """Add to a counter of either metrics flavour: this package's ``Metrics`` or any object
    with plain integer attributes, as the reference's harness passes."""
    if hasattr(metrics, "bump"):
        metrics.bump(name, value)
    else:
        setattr(metrics, name, int(getattr(metrics, name, 0)) + int(value))


def _mlp_weights(mod: Any) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    return mod.gate_proj.weight.detach(), mod.up_proj.weight.detach(), mod.down_proj.weight.detach()


def extract_experts(experts: Any) -> Tuple[str, List[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]]]:
    """Accept the two expert containers the reference accepts (:4350-4362): a fused object
    (``gate_up_proj [E,2I,H]``, ``down_proj [E,H,I]``) or a list of modules."""
    if hasattr(experts, "gate_up_proj") and hasattr(experts, "down_proj"):
        gu, dn = experts.gate_up_proj.detach(), experts.down_proj.detach()
        inter = gu.shape[1] // 2
        if not _is_silu(getattr(experts, "act_fn", None)):
            raise NotImplementedError("only SiLU experts are built")
        return "fused", [(gu[e, :inter], gu[e, inter:], dn[e]) for e in range(gu.shape[0])]
    try:
        mods = list(experts)
    except TypeError:
        mods = []
    if mods and all(hasattr(m, "gate_proj") and hasattr(m, "up_proj") and hasattr(m, "down_proj") for m in mods):
        for m in mods:
            if not _is_silu(getattr(m, "act_fn", None)):
                raise NotImplementedError("only SiLU experts are built")
        return "modulelist", [_mlp_weights(m) for m in mods]
    raise RuntimeError("Unsupported experts container. Need fused or modulelist experts.")


def quantized_experts(experts: Any, device: Any) -> List[Tuple[fp8.Quantized, fp8.Quantized, fp8.Quantized]]:
    """(values, scales) of every expert's gate, up and down: a module's own where it holds 8-bit weights with
    block scales, else quantised here, on ``device``."""
    kind, triples = extract_experts(experts)
    if kind == "modulelist":
        return [tuple(fp8.module_weight(m, device) for m in (e.gate_proj, e.up_proj, e.down_proj)) for e in experts]
    if any(w.dtype == fp8.E4M3 for w in triples[0]):
        raise NotImplementedError("fused containers of 8-bit experts are not built: give modules with weight_scale_inv")
    return [tuple(fp8.quantize_weight(w.to(device)) for w in t) for t in triples]


class _Workspace:
    """Activation buffers for one (T, layer shape); shared by all layers of that shape.  The
    most recently used ``SPARSE_HIP_WORKSPACE_CACHE`` (default 8) shapes are kept."""

    _cache = LruTable.from_env("SPARSE_HIP_WORKSPACE_CACHE", 8)

    def __init__(self, T: int, K: int, E: int, H: int, I: int, Is: int, dtype, logits_dtype, device,
                 weight_format: str = "native") -> None:
        self.logits_dtype = logits_dtype
        self.shared_gate = torch.empty((T,), device=device, dtype=dtype)
        self.topv = torch.empty((T, K), device=device, dtype=dtype)
        self.topi = torch.empty((T, K), device=device, dtype=torch.int64)
        self.perm = ops.Permutation(T, K, E, device)
        eight = weight_format == "fp8"       # the 8-bit products keep what they need in one block of bytes
        self.inter = None if eight else torch.empty((T * K, I), device=device, dtype=dtype)
        self.parts = torch.empty((T * K, H), device=device, dtype=dtype)
        self.shared_inter = torch.empty((T, Is), device=device, dtype=dtype) if Is and not eight else None
        self.fp8_ws = (torch.empty((fp8.moe_ffn_ws_bytes(T, K, E, min(E, T * K), H, I, Is),), device=device,
                                   dtype=torch.uint8) if eight else None)
        self.shared_out = torch.empty((T, H), device=device, dtype=dtype) if Is else None
        self.segs_dev = ops.seglist_device(self.perm, min(E, T * K))
        self.route_counter = torch.zeros((1,), device=device, dtype=torch.int32)
        # small decode calls cut the shared down projection's long reduction into parts (fp32
        # sums here) that the combine step finishes; from 17 tokens on the routed experts are
        # enough work beside it and the extra reads of the combine step cost more than they save
        self.split_parts = (ops.decode_split_parts(Is) if Is and T <= 16 and not eight
                            and dtype in ops.HALF_DTYPES and torch.device(device).type == "cuda" else 1)
        self.split_ws = ops.decode_split_workspace(T, H, device) if self.split_parts > 1 else None
        # host mirrors for the offloaded path (pinned, written by async D2H copies)
        self.host_offsets = torch.empty((E + 1,), dtype=torch.int32, pin_memory=True)
        self.host_rs_topi = torch.empty((T * E,), dtype=torch.int64, pin_memory=True)
        self.host_rs_topv = torch.empty((T * E,), dtype=torch.float32, pin_memory=True)

    @classmethod
    def get(cls, *key) -> "_Workspace":
        return cls._cache.get_or_make(key, lambda: cls(*key))


def _NO_SEGMENTS():
    return ops.seglist_host([], [])


class _EventRing:
    """Reusable events of one lane.  An event is only ever re-recorded on the same
    in-order lane, so waiting on a recycled event still implies the older work is done."""

    def __init__(self, n: int = 512) -> None:
        self._events = [ops.Event() for _ in range(n)]
        self._next = 0

    def take(self) -> ops.Event:
        ev = self._events[self._next]
        self._next = (self._next + 1) % len(self._events)
        return ev


class _SideStreams:
    """Upload streams shared by all layers (default priority)."""

    _inst: Optional["_SideStreams"] = None

    def __init__(self) -> None:
        self.prefetch = ops.SideStream()
        self.epipe = ops.SideStream()
        self.rings = {"compute": _EventRing(2048), "prefetch": _EventRing(2048), "epipe": _EventRing(512)}

    @classmethod
    def get(cls) -> "_SideStreams":
        if cls._inst is None:
            cls._inst = cls()
        return cls._inst


class _HipBackend(Backend):
    """Uploads, events and FFN launches for one layer's residency policy."""

    def __init__(self, block: "DistributedSparseMoeBlock") -> None:
        self.block = block
        self.streams = _SideStreams.get()
        self.rings = self.streams.rings
        self.x: Optional[torch.Tensor] = None
        self.ws: Optional[_Workspace] = None
        self.launches = 0

    def _stream(self, lane: str) -> int:
        if lane == "compute":
            return torch.cuda.current_stream().cuda_stream
        return self.streams.prefetch.handle if lane == "prefetch" else self.streams.epipe.handle

    def bind(self, x: torch.Tensor, ws: _Workspace) -> None:
        self.x, self.ws = x, ws

    def upload(self, eid: int, slot: int, lane: str):
        blk = self.block
        ev = self.rings[lane].take()
        stream = self._stream(lane)
        timed = blk.metrics.time_copies and len(blk.metrics.pending_events) < 100000
        if timed:
            start, end = ops.Event(timing=True), ops.Event(timing=True)
            start.record(stream)
        ops.expert_upload_async(blk.slab.slot_ptr(slot), blk.arena.host_ptr(eid), blk.arena.expert_bytes,
                                stream, ev)
        if timed:
            end.record(stream)
            stage = blk.residency.stage if blk.residency is not None else "none"
            blk.metrics.pending_events.append((start, end, f"{lane}_h2d_ms", blk.layer_idx, stage))
        return ev

    def event_done(self, event) -> bool:
        return event.query()

    def wait_event(self, event, lane: str, ordering: bool = False) -> None:
        event.wait(self._stream(lane))

    def run_segments(self, segments: Sequence[Tuple[int, int]]) -> None:
        blk, ws = self.block, self.ws
        segs = ops.seglist_host([e for e, _ in segments], [s for _, s in segments])
        if blk.weight_format == "fp8":
            fp8.moe_ffn(blk.slab, self.x, ws.topv, ws.perm, segs=segs, parts=ws.parts, ws=ws.fp8_ws)
        else:
            ops.grouped_swiglu(blk._experts_desc, self.x, ws.topv, ws.perm, segs, ws.inter, ws.parts)
        self.launches += 1

    def fence(self):
        ev = self.rings["compute"].take()
        ev.record(self._stream("compute"))
        return ev


class DistributedSparseMoeBlock(nn.Module):
    """Drop-in for the reference block on a single GPU (world size 1)."""

    def __init__(
        self,
        layer_idx: int,
        mlp_block: Any,
        scp_map: Any = None,
        env: Optional[DistEnv] = None,
        num_layers: int = 1,
        num_experts: Optional[int] = None,
        top_k: int = 1,
        dtype: torch.dtype = torch.bfloat16,
        expert_offload: str = "gpu",
        expert_cache: int = 10,
        routing_mode: str = "router",
        rs_dir: Optional[str] = None,
        rs_require_complete: bool = False,
        rs_prob_to_logit_eps: float = 1e-12,
        log_routing_stats: bool = False,
        rs_group: int = 3,
        rs_debug: bool = False,
        metrics: Optional[Metrics] = None,
        debug_a2a_checks: bool = False,
        collect_per_layer: bool = False,
        log_per_layer: bool = False,
        planner_mode: str = "none",
        prefetch_top_m: int = 1,
        oracle_mode: str = "none",
        oracle_ignore_cache_capacity: bool = True,
        placement_mode: str = "scp",
        expert_source: str = "router",
        cache_policy: str = "lru",
        runtime_mode: str = "baseline",
        topology: Any = None,
        residency_config: Optional[ResidencyConfig] = None,
        weight_format: str = "native",
    ) -> None:
        super().__init__()
        self.layer_idx = int(layer_idx)
        self.env = env if env is not None else DistEnv()
        self.device = torch.device(self.env.device)
        self.rank, self.world = int(self.env.rank), int(self.env.world)
        if self.world != 1:
            raise NotImplementedError("this build runs the MoE layer on one GPU (world size 1)")
        self.num_layers = int(num_layers)
        self.top_k = int(top_k)
        self.dtype = dtype
        # newer Hugging Face layouts keep the routing options on the router module
        gate_mod = getattr(mlp_block, "gate", None)
        self.norm_topk_prob = bool(getattr(mlp_block, "norm_topk_prob", getattr(gate_mod, "norm_topk_prob", False)))
        # None: the reference's rule (tensor only for the DeepSeek family, :9485-9488); a harness
        # sets it when the decoder layer it swaps into expects the other convention
        self.return_router_logits: Optional[bool] = None
        # enum validation, same messages as the reference (:4475-4498, :4799-4804)
        self.exec_routing_mode = str(routing_mode)
        if self.exec_routing_mode not in ("router", "rs"):
            raise ValueError(f"routing_mode must be router|rs, got {self.exec_routing_mode}")
        self.placement_mode = str(placement_mode)
        if self.placement_mode not in ("scp", "scp_ep", "round_robin", "weighted_random_balanced"):
            raise ValueError(
                f"placement_mode must be scp|scp_ep|round_robin|weighted_random_balanced, got {self.placement_mode}")
        self.planner_mode = str(planner_mode)
        if self.planner_mode not in ("none", "rs_prefetch"):
            raise ValueError(f"planner_mode must be none|rs_prefetch, got {self.planner_mode}")
        self.expert_source = str(expert_source)
        if self.expert_source not in ("router", "rs"):
            raise ValueError(f"expert_source must be router|rs, got {self.expert_source}")
        if str(runtime_mode) != "baseline":
            raise ValueError(f"Unsupported runtime_mode: {runtime_mode}")
        self.runtime_mode = "baseline"
        if self.expert_source == "rs" and not (self.exec_routing_mode == "rs" or self.planner_mode == "rs_prefetch"):
            raise ValueError(
                "expert_source=rs requires RS cache available, so routing_mode must be 'rs' "
                "or planner_mode must be 'rs_prefetch'.")
        # accepted by the reference, not built here: fail before any weight is touched
        if str(oracle_mode) != "none":
            raise NotImplementedError(f"oracle_mode={oracle_mode} (record / replay traces) is not built")
        self.oracle_mode = "none"
        self.expert_offload = str(expert_offload)
        # Read and validated as the reference does (:4795-4798).  Both settings are satisfied by
        # construction here: "fixed64" asks for a prefill summation order that does not depend on where a
        # row sits in its expert's batch or on how many rows that batch has, per-row decode granularity for
        # the same of a decode call -- the prefill-size kernels and the decode-size kernels each reduce every
        # output element over k in one fixed order (64-wide slabs in sequence, the same MFMA sequence inside
        # a slab), whatever the row's position and whoever shares its tile.
        self._native_decode_granularity = str(os.environ.get("SPARSE_EP_NATIVE_DECODE_GRANULARITY", "0")).strip().lower() \
            not in ("0", "false", "no", "off")
        self._prefill_expert_math = str(os.environ.get("SPARSE_PREFILL_EXPERT_MATH", "native")).strip().lower()
        if self._prefill_expert_math not in ("native", "fixed64"):
            raise ValueError("SPARSE_PREFILL_EXPERT_MATH must be native or fixed64")
        if self.expert_offload not in ("cpu", "gpu"):
            raise ValueError(f"expert_offload must be cpu|gpu, got {self.expert_offload}")
        self.cache_policy = str(cache_policy).lower()
        if self.cache_policy not in ("lru", "lfu", "tiered"):
            raise ValueError(f"cache_policy must be lru|lfu|tiered, got {self.cache_policy}")
        if self.dtype not in (torch.bfloat16, torch.float16, torch.float32):
            raise ValueError(f"dtype must be bfloat16, float16 or float32, got {self.dtype}")
        # "native": expert weights in `dtype`; "fp8": in 8 bits with a scale per 128 x 128 block (the reference
        # has no such path)
        self.weight_format = str(weight_format).lower()
        if self.weight_format not in ("native", "fp8"):
            raise ValueError(f"weight_format must be native|fp8, got {weight_format}")
        if self.weight_format == "fp8" and self.dtype not in ops.HALF_DTYPES:
            raise ValueError(f"weight_format=fp8 needs bfloat16 or float16 activations, got {self.dtype}")
        self.rs_group = int(rs_group)
        self.rs_prob_to_logit_eps = float(rs_prob_to_logit_eps)
        self.prefetch_top_m = int(prefetch_top_m)
        self.metrics = metrics if metrics is not None else Metrics()
        # all-resident decode calls of up to 16 tokens: combine inside the down projection's launch
        # (SPARSE_HIP_FOLD_COMBINE=0 keeps the separate combine launch; same bits either way)
        self.route_with_shared = str(os.environ.get("SPARSE_HIP_ROUTE_WITH_SHARED", "1")).strip().lower() not in (
            "0", "false", "no", "off")
        self._shared_up_wanted = False      # forward: the call's expert launches can take a ready shared_inter
        self._shared_inter_ready = False    # _route: this call's routing launch has filled it
        self.fold_combine = str(os.environ.get("SPARSE_HIP_FOLD_COMBINE", "1")).strip().lower() not in (
            "", "0", "false", "no", "off")
        # all-resident prefill-size batches run routed and shared tiles in one launch per projection
        # (SPARSE_HIP_MERGED_PREFILL=0: separate launches; same bits either way)
        self.merged_prefill = str(os.environ.get("SPARSE_HIP_MERGED_PREFILL", "1")).strip().lower() not in (
            "", "0", "false", "no", "off")
        # ... and otherwise the shared expert on a second stream beside the routing
        self.overlap_shared = str(os.environ.get("SPARSE_HIP_OVERLAP_SHARED", "1")).strip().lower() not in (
            "", "0", "false", "no", "off")

        # ---- weights --------------------------------------------------------
        if not hasattr(mlp_block, "gate") or not hasattr(mlp_block, "experts"):
            raise RuntimeError("mlp_block needs .gate and .experts")
        self.moe_family = "qwen_shared" if hasattr(mlp_block, "shared_expert") else "deepseek_shared"
        self.routed_scaling_factor = float(getattr(mlp_block.gate, "routed_scaling_factor",
                                                   getattr(mlp_block, "routed_scaling_factor", 1.0)) or 1.0)
        self.gate_weight = mlp_block.gate.weight.detach().to(self.device, self.dtype).contiguous()
        # selection method of a DeepSeek-family gate module (the reference runs whatever gate the
        # model brings, :9503-9517): plain greedy top-k, or limited to the best expert groups
        bias = getattr(gate_mod, "e_score_correction_bias", None)
        method = str(getattr(gate_mod, "topk_method", None) or ("greedy" if bias is None else "noaux_tc"))
        if method not in ("greedy", "group_limited_greedy", "noaux_tc"):
            raise NotImplementedError(f"gate topk_method={method} is not built (greedy | group_limited_greedy | noaux_tc)")
        if (method == "noaux_tc") != (bias is not None):
            raise ValueError("gate topk_method=noaux_tc goes with e_score_correction_bias")
        # a gate balanced by a bias ranks the sigmoid of the logits plus the bias, groups by their two best
        self.gate_score = str(getattr(gate_mod, "scoring_func", None) or ("softmax" if bias is None else "sigmoid"))
        if self.gate_score not in ops.SELECT_SCORE:
            raise NotImplementedError(f"gate scoring_func={self.gate_score} is not built (softmax | sigmoid)")
        self.gate_bias = None if bias is None else bias.detach().to(self.device, torch.float32).reshape(-1).contiguous()
        self.gate_group_score = "max" if bias is None else "top2"
        self.n_group = self.topk_group = 1
        if method != "greedy":
            self.n_group = int(getattr(gate_mod, "num_group", None) or getattr(gate_mod, "n_group", None) or 1)
            self.topk_group = int(getattr(gate_mod, "topk_group", None) or self.n_group)
            if self.topk_group >= self.n_group:
                self.n_group = self.topk_group = 1          # every group kept: plain top-k
        self.experts_kind, expert_weights = extract_experts(mlp_block.experts)
        if self.weight_format != "fp8" and any(w.dtype == fp8.E4M3 for triple in expert_weights for w in triple):
            raise ValueError("8-bit expert weights need weight_format='fp8'")
        self.num_experts = int(num_experts) if num_experts is not None else len(expert_weights)
        if self.num_experts != len(expert_weights) or self.gate_weight.shape[0] != self.num_experts:
            raise ValueError("num_experts does not match the gate / experts container")
        self.hidden_size = int(self.gate_weight.shape[1])
        self.inter_size = int(expert_weights[0][0].shape[0])
        shared_mod = getattr(mlp_block, "shared_expert", None) or getattr(mlp_block, "shared_experts", None)
        self.shared_weights = None
        self.shared_inter_size = 0
        if shared_mod is not None:
            if not _is_silu(getattr(shared_mod, "act_fn", None)):
                raise NotImplementedError("only SiLU shared experts are built")
            if self.weight_format == "fp8":
                self.shared_weights = tuple(
                    fp8.Weight.from_quantized(*fp8.module_weight(m, self.device))
                    for m in (shared_mod.gate_proj, shared_mod.up_proj, shared_mod.down_proj))
            else:
                if any(w.dtype == fp8.E4M3 for w in _mlp_weights(shared_mod)):
                    raise ValueError("8-bit shared-expert weights need weight_format='fp8'")
                # tiled content, logical [rows, cols] shape kept for argument checks
                self.shared_weights = tuple(
                    tile_weight(t.to(self.device, self.dtype)).reshape(t.shape).contiguous()
                    for t in _mlp_weights(shared_mod))
            self.shared_inter_size = int(self.shared_weights[0].shape[0])
        sg = getattr(mlp_block, "shared_expert_gate", None)
        self.shared_gate_weight = (
            sg.weight.detach().to(self.device, self.dtype).reshape(-1).contiguous() if sg is not None else None)
        self.logits_dtype = torch.float32 if self.moe_family == "deepseek_shared" else self.dtype
        # decode-size batches route on a packed copy of the gate (and shared gate) rows where
        # the shapes allow it; everything else reads the row-major weights
        self.gate_packed = ops.pack_router_gate(self.gate_weight, self.shared_gate_weight)

        E, H, I = self.num_experts, self.hidden_size, self.inter_size
        self.local_expert_ids = list(range(E))
        self._local_eid_set = set(self.local_expert_ids)
        self.residency: Optional[LayerResidency] = None
        self.arena: Optional[HostExpertArena] = None
        eight = self.weight_format == "fp8"
        if self.expert_offload == "gpu":
            self.slab = (fp8.ExpertSlab.from_quantized(quantized_experts(mlp_block.experts, self.device), self.device)
                         if eight else ExpertSlab.resident(expert_weights, H, I, self.dtype, self.device))
        else:
            cfg = residency_config if residency_config is not None else ResidencyConfig.from_env(
                capacity=int(expert_cache), planner_mode=self.planner_mode, prefetch_top_m=int(prefetch_top_m))
            cfg.capacity = int(expert_cache) if residency_config is None else cfg.capacity
            if residency_config is None:
                cfg.cache_policy = self.cache_policy
            elif cfg.cache_policy != self.cache_policy and self.cache_policy != "lru":
                cfg.cache_policy = self.cache_policy
            self.arena = (fp8.HostExpertArena(quantized_experts(mlp_block.experts, self.device), H, I, pin=True)
                          if eight else HostExpertArena(expert_weights, H, I, self.dtype, pin=True))
            self._backend = _HipBackend(self)
            self.residency = LayerResidency(self.layer_idx, E, self.top_k, cfg, self._backend, self.metrics,
                                            expert_bytes=self.arena.expert_bytes)
            self.slab = (fp8.ExpertSlab(self.residency.num_slots, E, H, I, self.device) if eight
                         else ExpertSlab(self.residency.num_slots, E, H, I, self.dtype, self.device))
        self._experts_desc = None if eight else ops.make_experts(self.slab.data, self.slab.expert_slot, E, H, I)
        self._cache = self.residency.cache if self.residency is not None else None
        self._current_forward_batch_size = 0
        self._current_forward_seq_len = 0
        SparseContext.register_layer_block(self.layer_idx, self)

    # ------------------------------------------------------------------ helpers
    def _return_tensor_only_mlp(self) -> bool:
        if self.return_router_logits is not None:
            return not self.return_router_logits
        return self.moe_family == "deepseek_shared"

    def _current_stage(self, seq_len: Optional[int] = None) -> str:
        """Reference :6149-6158."""
        phase = str(SparseContext.current_phase or "none").strip().lower()
        if phase in ("prefill", "decode"):
            return phase
        seq = int(seq_len) if seq_len is not None else int(self._current_forward_seq_len or 0)
        if seq > 0:
            return "decode" if seq == 1 else "prefill"
        return "decode"

    def _workspace(self, T: int, K: Optional[int] = None) -> _Workspace:
        return _Workspace.get(T, self.top_k if K is None else int(K), self.num_experts, self.hidden_size,
                              self.inter_size,
                              self.shared_inter_size, self.dtype, self.logits_dtype, self.device,
                              *(() if self.weight_format == "native" else (self.weight_format,)))

    _shared_streams: dict = {}

    def _shared_stream(self) -> "torch.cuda.Stream":
        """The stream (default priority, one per device) the shared expert of prefill-size
        batches runs on."""
        key = (self.device.type, self.device.index)
        st = DistributedSparseMoeBlock._shared_streams.get(key)
        if st is None:
            st = torch.cuda.Stream(device=self.device)
            DistributedSparseMoeBlock._shared_streams[key] = st
        return st

    # ------------------------------------------------------------------ segment timing
    def _segment_timing_on(self) -> bool:
        """``SPARSE_EXPERT_TIMING=1``, read per call like the reference does (:14656)."""
        return self.metrics is not None and os.environ.get("SPARSE_EXPERT_TIMING", "0").strip().lower() in (
            "1", "true", "yes", "on")

    def _timed_segment(self, name: str, fn, on: Optional[bool] = None):
        """``_timed_segment`` (utils/eval_core.py:14655-14676): the segment between two events
        on the compute stream, waited for at once, added to ``metrics.moe_<name>_ms``.  Timing
        serialises the layer, so the block runs its one-stream, one-kernel-per-segment form
        while it is on; the values do not change."""
        if not (self._segment_timing_on() if on is None else on):
            return fn()
        start, end = ops.Event(timing=True), ops.Event(timing=True)
        start.record()
        out = fn()
        end.record()
        torch.cuda.current_stream().synchronize()
        field = {"router": "moe_router_ms", "expert": "moe_expert_ms", "shared": "moe_shared_ms"}[name]
        setattr(self.metrics, field, float(getattr(self.metrics, field, 0.0)) + start.elapsed_ms(end))
        self.metrics.moe_timing_calls = int(getattr(self.metrics, "moe_timing_calls", 0)) + 1
        return out

    # ------------------------------------------------------------------ routing
    def _route(self, x: torch.Tensor, ws: _Workspace, after_logits=None) -> torch.Tensor:
        """Router logits (+ shared gate), fused softmax/top-k, permutation (:9519-9595).
        Returns the logits, a fresh tensor the caller owns.  ``after_logits`` is called once
        the logits (and the shared gate) are queued: the point from which the shared expert
        no longer depends on anything the rest of the routing does."""
        after_logits = after_logits or (lambda: None)
        logits = torch.empty((x.shape[0], self.num_experts), device=x.device, dtype=self.logits_dtype)
        shared_gate = ws.shared_gate if self.shared_gate_weight is not None else None
        selects = self.gate_bias is not None or self.gate_score != "softmax"
        one_launch = self.routed_scaling_factor == 1.0 and self.n_group == 1 and not selects
        if self.gate_packed is not None and x.shape[0] <= ops.ROUTE_PACKED_MAX_TOKENS and one_launch:
            # the routing launch also runs the shared expert's gate and up projections where it can
            beside = self._shared_up_wanted
            ops.route_decode_packed(x, self.gate_packed, self.num_experts, self.shared_gate_weight is not None,
                                    self.top_k, self.norm_topk_prob, logits, shared_gate, ws.topv, ws.topi, ws.perm,
                                    shared_up=(self.shared_weights[0], self.shared_weights[1], ws.shared_inter)
                                    if beside else None)
            self._shared_inter_ready = bool(beside)
            after_logits()
            return logits
        if x.shape[0] <= ops.DECODE_MAX_TOKENS and one_launch:
            ops.route_decode(x, self.gate_weight, self.shared_gate_weight, self.top_k, self.norm_topk_prob, logits,
                             shared_gate, ws.topv, ws.topi, ws.perm, ws.route_counter)
            after_logits()
            return logits
        ops.router_logits(x, self.gate_weight, self.shared_gate_weight, self.logits_dtype, out=logits,
                          shared_gate_out=shared_gate)
        after_logits()
        if selects:
            ops.gate_select(logits, self.top_k, self.gate_score, self.gate_bias, self.n_group, self.topk_group,
                            self.gate_group_score, self.norm_topk_prob, self.routed_scaling_factor, self.dtype,
                            topv=ws.topv, topi=ws.topi)
            ops.permute_build(ws.topi, self.num_experts, out=ws.perm)
            return logits
        # the routed scaling factor multiplies in fp32 inside the top-k launch, before the one rounding to
        # the activation dtype, as the gate module does before the reference's cast (:9509-9513)
        ops.gate_topk(logits, self.top_k, self.norm_topk_prob, out_dtype=self.dtype, topv=ws.topv, topi=ws.topi,
                      n_group=self.n_group, topk_group=self.topk_group, scale=self.routed_scaling_factor)
        ops.permute_build(ws.topi, self.num_experts, out=ws.perm)
        return logits

    def _route_from_cache(self, x: torch.Tensor, ws: _Workspace) -> torch.Tensor:
        """``expert_source="rs"``: execute with the weights and indices the previous layer's
        predictor left in ``SparseContext.routing_cache`` (:11118-11155).  Returns pseudo
        logits: log of the replayed weight at the chosen experts, -1e9 elsewhere."""
        w, idx = SparseContext.routing_cache[self.layer_idx]
        T = int(x.shape[0])
        if tuple(idx.shape) != tuple(ws.topi.shape) or tuple(w.shape) != tuple(ws.topv.shape):
            raise RuntimeError(f"cached routing of shape {tuple(idx.shape)} does not fit {T} tokens")
        ws.topv.copy_(w.to(self.dtype))
        ws.topi.copy_(idx)
        ops.permute_build(ws.topi, self.num_experts, out=ws.perm)
        if self.shared_gate_weight is not None:
            # the shared expert's gate comes out of the router-logits kernel; the logits are unused
            ops.router_logits(x, self.gate_weight, self.shared_gate_weight, self.logits_dtype,
                              shared_gate_out=ws.shared_gate)
        return ops.pseudo_logits(ws.topv, ws.topi, self.num_experts, eps=self.rs_prob_to_logit_eps, fill=-1e9)

    def _routing_router(self, x: torch.Tensor):
        """``(topv, topi, router_logits)`` like the reference's method (:9502-9595)."""
        ws = self._workspace(int(x.shape[0]))
        logits = self._route(x.contiguous(), ws)
        if self.moe_family == "deepseek_shared":
            logits = ops.pseudo_logits(ws.topv, ws.topi, self.num_experts, eps=1e-12, fill=float("-inf"))
        return ws.topv, ws.topi, logits

    # ------------------------------------------------------------------ RS prefetch
    def _next_layer_rs_feature_mode(self) -> str:
        """What the predictor of the next layer reads (:10910-10914)."""
        target = self.layer_idx + 1
        if SparseContext.rs_bank is None or target >= len(SparseContext.rs_bank):
            return "hidden"
        return str(getattr(SparseContext.rs_bank[target], "rs_feature_mode", "hidden"))

    def _rs_begin(self, x: torch.Tensor, seq_len: int, ws: _Workspace, source=None):
        """Device half of ``_compute_and_schedule_next_layer_rs`` (:10916-11010): budget on
        the host, predictor + top-k on the device, async copy of the top-k to the host.
        ``source`` = this layer's own (ids, weights) for predictors that read them."""
        for_routing = self.expert_source == "rs" or self.exec_routing_mode == "rs"
        if (self.planner_mode != "rs_prefetch" and not for_routing) or SparseContext.rs_bank is None:
            return None
        if SparseContext.rs_bank_layout != "next_layer":
            return None
        target = self.layer_idx + 1
        if target >= self.num_layers:
            return None
        src = SparseContext.rs_bank_source_layers
        if target >= len(src) or int(src[target]) != self.layer_idx:
            return None
        tblk = SparseContext.layer_blocks.get(target)
        if tblk is None or target >= len(SparseContext.rs_bank):
            return None
        tres = tblk.residency
        if int(seq_len) != 1 and not (tres is not None and tres.cfg.rs_prefetch_prefill):
            return None
        budget = 0
        if self.planner_mode == "rs_prefetch" and tres is not None:
            tres.phase, tres.call_id = str(SparseContext.current_phase), int(SparseContext.runtime_call_id)
            key = ("next_layer_rs", str(SparseContext.current_phase), int(SparseContext.runtime_call_id),
                   self.layer_idx, target)
            budget = tres.prefetch_budget(key)
        if budget <= 0 and not for_routing:
            return None
        if tres is not None and tres.light_policy is not None:
            # time a copy issued now has before its layer runs: this layer's routed compute
            # plus the next attention (reference :10993-10996)
            policy = tres.light_policy
            here = policy.profile.cost(self.rank, self.layer_idx)
            policy.window_ms = here.compute(self.top_k, int(x.shape[0]) * self.top_k) + policy.cost.attention
        mode = self._next_layer_rs_feature_mode()
        module = SparseContext.rs_bank[target]
        if mode not in ("hidden", "hidden_router_topk"):
            raise RuntimeError(f"Unsupported next-layer RS feature_mode={mode}")
        if mode == "hidden_router_topk" and source is None:
            return None
        fused = fused_scout(module, x, mode, self.num_experts)
        if fused is not None:
            # HIP predictor on the token rows as they are (after one launch that appends the routing
            # columns, for predictors that read them)
            pred = fused(x if mode == "hidden" else ops.rs_features(x, source[0], source[1], self.num_experts))
        else:
            rs_in = x.float()
            if mode == "hidden_router_topk":
                rs_in = torch.cat([rs_in, router_topk_feature(source[0], source[1], self.num_experts)], dim=-1)
            pred = module(rs_in).to(torch.float32)
        self.metrics.rs_next_layer_pred_calls += 1
        self.metrics.rs_mlp_calls += 1
        if for_routing:
            # the next layer may execute with this prediction instead of its router (:10971-10983)
            raw = os.environ.get("SPARSE_RS_EXEC_TOPK", "").strip()
            exec_topk = max(1, min(int(raw) if raw else self.top_k, int(pred.shape[-1])))
            route_v, route_i = stable_topk(pred, exec_topk)
            if self.norm_topk_prob:
                route_v = route_v / route_v.sum(dim=-1, keepdim=True).clamp_min(1e-12)
            SparseContext.routing_cache[target] = (route_v.to(x.dtype), route_i.to(torch.long))
        if self.planner_mode != "rs_prefetch" or tres is None or budget <= 0:
            return None
        topi, topv = topk_for_planning(pred, tres.predict_topk(), self.norm_topk_prob, x.dtype)
        T, pred_k = int(topi.shape[0]), int(topi.shape[1])
        ws.host_rs_topi[:T * pred_k].view(T, pred_k).copy_(topi, non_blocking=True)
        ws.host_rs_topv[:T * pred_k].view(T, pred_k).copy_(topv, non_blocking=True)
        return (tres, budget, T, pred_k)

    def _rs_finish(self, job, ws: _Workspace) -> None:
        """Host half: score, plan, admit; uploads go to the prefetch stream."""
        tres, budget, T, pred_k = job
        ids = ws.host_rs_topi[:T * pred_k].tolist()
        probs = ws.host_rs_topv[:T * pred_k].tolist()
        if self.metrics.events is not None:
            self.metrics.bump("rs_plans")
        plan = tres.schedule_prefetch(ids, probs, budget)
        hook = getattr(self, "_rs_plan_hook", None)
        if hook is not None:
            hook(self.layer_idx, ids, probs, budget, plan)

    # ------------------------------------------------------------------ forward
    @torch.no_grad()
    def forward(self, hidden_states: torch.Tensor):
        if hidden_states.dim() != 3:
            raise ValueError("hidden_states must be [B, S, H]")
        B, S, H = hidden_states.shape
        if H != self.hidden_size:
            raise ValueError(f"hidden size {H} does not match the layer's {self.hidden_size}")
        if hidden_states.dtype != self.dtype:
            raise ValueError(f"hidden_states must be {self.dtype}, got {hidden_states.dtype}")
        x = hidden_states.view(-1, H)
        T = int(x.shape[0])
        self._current_forward_batch_size, self._current_forward_seq_len = int(B), int(S)
        SparseContext.current_moe_layer_idx = self.layer_idx
        if T == 0:
            logits = torch.empty((0, self.num_experts), device=x.device, dtype=self.logits_dtype)
            return hidden_states if self._return_tensor_only_mlp() else (hidden_states, logits)
        # a layer that replays its predecessor's prediction executes as many experts per token as
        # that prediction holds (SPARSE_RS_EXEC_TOPK, :10979-10987), not necessarily its own top-k
        from_cache = self.expert_source == "rs" and self.layer_idx in SparseContext.routing_cache
        k_exec = int(SparseContext.routing_cache[self.layer_idx][1].shape[-1]) if from_cache else self.top_k
        ws = self._workspace(T, k_exec)
        staging = SparseContext.staging
        staged = (staging is not None and self.residency is not None and staging.handles(self, S))
        if staged:
            # forecast staging: the prediction for layer l+1 leaves on a side stream and is never
            # joined; this layer's own ring window is sealed at the executor
            self.residency.staging = staging
            staging.forecast_next(self, x, int(SparseContext.runtime_call_id))
            rs_job = None
        else:
            if self.residency is not None:
                self.residency.staging = None
            # a predictor that also reads this layer's routing runs after it (:16466-16506)
            rs_job = self._rs_begin(x, S, ws) if self._next_layer_rs_feature_mode() == "hidden" else None

        shared_gate = ws.shared_gate if self.shared_gate_weight is not None else None
        timing = self._segment_timing_on()
        eight = self.weight_format == "fp8"
        fused = (not eight and self.residency is None and self.shared_weights is not None and self.dtype in ops.HALF_DTYPES
                 and T <= ops.DECODE_MAX_TOKENS and not timing)
        # Prefill-size batches: the shared expert needs only x and the shared gate, so it runs
        # on a second stream from the moment the logits kernel is queued, beside top-k,
        # permutation, tile map and the first routed tiles, and is joined before combine.
        merged = (self.merged_prefill and not eight and self.residency is None and self.dtype in ops.HALF_DTYPES and x.is_cuda
                  and T > ops.DECODE_MAX_TOKENS and not timing)
        side = (self._shared_stream() if self.shared_weights is not None and not fused and self.overlap_shared
                and x.is_cuda and T > ops.DECODE_MAX_TOKENS and not timing and not merged and not eight else None)

        # Whether the shared expert's down projection is left as partial sums for the combine
        # step depends on the call's size and dtype only, never on where the routed experts
        # live: an offloaded layer must give the bits of the all-resident one.
        split_shared = self.shared_weights is not None and ws.split_ws is not None
        # Calls of up to 16 tokens compute the shared expert's gate and up projections with the
        # 16-wavefront kernel, beside the routing when this call routes with the packed router,
        # alone otherwise: the same code, so the same bits, wherever it runs.
        shared_up_alone = (self.shared_weights is not None and not eight and self.dtype in ops.HALF_DTYPES and x.is_cuda
                           and self.route_with_shared and T <= ops.ROUTE_PACKED_MAX_TOKENS
                           and self.shared_inter_size % 32 == 0 and H % 64 == 0)
        self._shared_up_wanted = shared_up_alone and not timing
        self._shared_inter_ready = False

        def shared_inter_ready() -> bool:
            if shared_up_alone and not self._shared_inter_ready:
                ops.shared_gate_up(x, self.shared_weights[0], self.shared_weights[1], ws.shared_inter)
                self._shared_inter_ready = True
            return self._shared_inter_ready

        def run_shared() -> None:
            if self.shared_weights is None or fused or merged:
                return
            if eight:
                # beside the routed experts in their launches, unless those are executed or timed apart
                if self.residency is not None or timing:
                    fp8.moe_ffn(self.slab, x, ws.topv, ws.perm, shared=self.shared_weights, shared_gate=shared_gate,
                                segs=_NO_SEGMENTS(), parts=ws.parts, shared_out=ws.shared_out, ws=ws.fp8_ws)
                return
            gw, uw, dw = self.shared_weights
            if split_shared:
                # the fused decode entry point with no routed segment: the shared expert alone,
                # in the same split form the all-resident call uses
                ops.moe_ffn_decode(self._experts_desc, x, ws.topv, ws.perm, _NO_SEGMENTS(), ws.inter, ws.parts,
                                   self.shared_weights, shared_gate, ws.shared_inter, ws.shared_out, ws.split_ws,
                                   shared_inter_ready=shared_inter_ready())
                return
            if side is None:
                ops.shared_expert(x, gw, uw, dw, shared_gate, ws.shared_inter, ws.shared_out,
                                  inter_ready=shared_inter_ready())
                return
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                ops.shared_expert(x, gw, uw, dw, shared_gate, ws.shared_inter, ws.shared_out)

        if timing:
            # router, then (below) routed experts, then the shared expert: the reference's order
            logits = self._timed_segment("router", lambda: (self._route_from_cache(x, ws) if from_cache
                                                            else self._route(x, ws)), on=True)
        elif from_cache:
            logits = self._route_from_cache(x, ws)
            run_shared()
        else:
            # also the first layer and prefill of an RS-routed run (:11128-11136)
            logits = self._route(x, ws, after_logits=run_shared)
        if not staged and self._next_layer_rs_feature_mode() == "hidden_router_topk":
            rs_job = self._rs_begin(x, S, ws, source=(ws.topi, ws.topv))

        out = torch.empty((T, H), device=x.device, dtype=self.dtype)
        combined = False

        def run_experts() -> None:
            nonlocal combined, rs_job
            if fused and split_shared and self.fold_combine:
                # small decode call, everything resident: the down projection's launch also combines
                ops.moe_ffn_decode_combine(self._experts_desc, x, ws.topv, ws.perm, ws.segs_dev, ws.inter, ws.parts,
                                           self.shared_weights, shared_gate, ws.shared_inter, ws.split_ws, out,
                                           shared_inter_ready=shared_inter_ready())
                combined = True
            elif fused:
                ops.moe_ffn_decode(self._experts_desc, x, ws.topv, ws.perm, ws.segs_dev, ws.inter, ws.parts,
                                   self.shared_weights, shared_gate, ws.shared_inter, ws.shared_out, ws.split_ws,
                                   shared_inter_ready=shared_inter_ready())
            elif merged:
                ops.moe_ffn_prefill(self._experts_desc, x, ws.topv, ws.perm, ws.segs_dev, ws.inter, ws.parts,
                                    self.shared_weights, shared_gate, ws.shared_inter, ws.shared_out)
            elif self.residency is None and eight:
                fp8.moe_ffn(self.slab, x, ws.topv, ws.perm, shared=None if timing else self.shared_weights,
                            shared_gate=shared_gate, segs=ws.segs_dev, parts=ws.parts, shared_out=ws.shared_out, ws=ws.fp8_ws)
            elif self.residency is None:
                ops.grouped_swiglu(self._experts_desc, x, ws.topv, ws.perm, ws.segs_dev, ws.inter, ws.parts)
            else:
                ws.host_offsets.copy_(ws.perm.seg_offsets, non_blocking=True)
                torch.cuda.current_stream().synchronize()
                if rs_job is not None:
                    self._rs_finish(rs_job, ws)
                off = ws.host_offsets.tolist()
                segments = [(e, off[e + 1] - off[e]) for e in range(self.num_experts) if off[e + 1] > off[e]]
                res = self.residency
                res.phase, res.call_id = str(SparseContext.current_phase), int(SparseContext.runtime_call_id)
                res.stage = self._current_stage(S)
                self._backend.bind(x, ws)
                if staged:
                    staging.seal(self, int(SparseContext.runtime_call_id))
                try:
                    self.last_executor = res.execute(segments)
                finally:
                    if staged:
                        staging.settle(self)

        self._timed_segment("expert", run_experts, on=timing)
        if timing:
            self._timed_segment("shared", run_shared, on=True)
        if self.residency is None and rs_job is not None:
            torch.cuda.current_stream().synchronize()
            self._rs_finish(rs_job, ws)

        if side is not None:
            torch.cuda.current_stream().wait_stream(side)
        if combined:
            pass
        elif split_shared:
            ops.combine_split(ws.parts, ws.perm, ws.split_ws, ws.split_parts, shared_gate, T, k_exec, out)
        else:
            ops.combine(ws.parts, ws.perm, ws.shared_out, T, k_exec, out)
        out = out.view(B, S, H)
        if self._return_tensor_only_mlp():
            return out
        return out, logits

    # ------------------------------------------------------------------ lifecycle hooks
    def _finalize_prev_group_prefetch(self) -> None:
        if self.residency is not None:
            self.residency.finalize_prev_group_prefetch()

    def reset_runtime_state_for_new_request(self, *, clear_expert_cache: bool = False,
                                            clear_cache_metadata: bool = True, demote_hot: bool = False) -> None:
        """Reference :6097-6147."""
        if self.residency is not None:
            self.residency.reset_for_new_request(clear_expert_cache=clear_expert_cache,
                                                 clear_cache_metadata=clear_cache_metadata)

    @classmethod
    def clear_all_expert_caches(cls) -> None:
        for blk in SparseContext.layer_blocks.values():
            if blk.residency is not None:
                blk.residency.clear()

    @classmethod
    def demote_prefill_scp_transients_for_decode(cls, metrics: Optional[Any] = None) -> None:
        """Once per request, at the prefill -> decode boundary (:16629-16653): entries that
        EPIPE staged and committed during prefill go to the LRU end of their cache."""
        if SparseContext.prefill_scp_transient_demoted_for_decode:
            return
        resident = demoted = 0
        for blk in list(SparseContext.layer_blocks.values()):
            cache = getattr(blk, "_cache", None)
            if cache is None:
                continue
            resident += len(cache.prefill_scp_transient_ids())
            demoted += int(cache.demote_prefill_scp_transients())
        if metrics is not None:
            _bump(metrics, "prefill_scp_transient_resident_at_decode_start", resident)
            _bump(metrics, "prefill_scp_transient_demote_count", demoted)
            _bump(metrics, "epipe_prefill_transient_demote_count", demoted)
        SparseContext.prefill_scp_transient_demoted_for_decode = True

    @classmethod
    def record_prefill_scp_transient_decode_end(cls, metrics: Optional[Any] = None) -> None:
        """Transient entries still resident when decoding ends (:16655-16667)."""
        if metrics is None:
            return
        left = 0
        for blk in list(SparseContext.layer_blocks.values()):
            cache = getattr(blk, "_cache", None)
            if cache is not None:
                left += len(cache.prefill_scp_transient_ids())
        _bump(metrics, "prefill_scp_transient_resident_at_decode_end", left)

    @classmethod
    def handle_epipe_prefill_extra_cache_decode_boundary(cls, metrics: Optional[Any] = None) -> None:
        """Count the payloads the prefill side caches hold at the boundary and drop them only
        where ``SPARSE_EPIPE_PREFILL_EXTRA_CACHE_CLEAR_AT_DECODE`` asks for it (:16591-16610);
        by default decode keeps reading them."""
        held = cleared = 0
        for blk in list(SparseContext.layer_blocks.values()):
            res = getattr(blk, "residency", None)
            if res is None:
                continue
            held += res.extra_cache.resident_count()
            if res.cfg.epipe_prefill_extra_cache_clear_at_decode:
                res.flush()
                cleared += res.clear_extra_cache()
        if metrics is not None:
            _bump(metrics, "epipe_prefill_extra_cache_resident_at_decode_start", held)
            if cleared > 0:
                _bump(metrics, "epipe_prefill_extra_cache_evict_count", cleared)

    @classmethod
    def record_epipe_prefill_extra_cache_decode_end(cls, metrics: Optional[Any] = None) -> None:
        """:16612-16627."""
        if metrics is None:
            return
        held = sum(blk.residency.extra_cache.resident_count() for blk in list(SparseContext.layer_blocks.values())
                   if getattr(blk, "residency", None) is not None)
        _bump(metrics, "epipe_prefill_extra_cache_resident_count", held)
        _bump(metrics, "epipe_prefill_extra_cache_resident_at_decode_end", held)
