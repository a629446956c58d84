"""Base sparse-MoE block over packed experts, backed by the sm_100a library.

Keeps the module interface of ``bitsmoe.models.base_block.BitsMoE_BaseSparseMoeBlock``
(bitsmoe/models/base_block.py:9-446): the three persistent fp16 shared-basis buffers,
``set_shared_basis`` / ``set_expert`` / ``set_super_expert_projected_weights`` /
``prepare_runtime_fastpath``, the lazily built runtime cache with its ``_*_static`` tuples and
``_packed_global_to_local`` map, ``_build_packed_routing``, ``_run_super_experts``,
``_packed_forward_cuda`` / ``_packed_forward_grouped`` at the reference's op boundary.

What differs is where the work happens: the cache also owns a ``PackedLayer`` (device pointer
tables built once per block), routing is built by one kernel without a device->host sync, and
``_fused_forward`` runs route -> basis -> experts -> down basis (+ residual) on one stream.
"""
from __future__ import annotations

import threading
from typing import Dict, List, Optional, Sequence, Tuple

import torch
import torch.nn as nn

from bitsmoe_b200.algorithms import _HAS_MLP_FORWARD_CUDA, mlp_forward_cuda
from bitsmoe_b200.models.swiglu import runs_as_swiglu
from bitsmoe_b200.quant.linear4 import Linear4

_FIELDS = ("payload", "rank_idx", "tile_meta", "slab_meta", "scale", "s")
_TAGS = ("gate", "up", "down")
_STACKING: Dict[torch.device, threading.Lock] = {}


def _stacking_lock(device: torch.device) -> threading.Lock:
    """Of all blocks on a device: an expert may belong to several blocks, and a block is copied and pickled without it.  Not of all devices: who
    holds it waits for its device, whose work may wait for a collective that the thread of another device has yet to launch."""
    return _STACKING.setdefault(device, threading.Lock())



class BitsMoE_BaseSparseMoeBlock(nn.Module):
    _SHARED_BASIS_BUFFER_KEYS = ("shared_vh_gate_proj", "shared_vh_up_proj", "shared_u_down")

    def _init_bitsmoe_common_state(self, super_experts: Optional[List[int]] = None,
                                   track_super_projected_weights: bool = False) -> None:
        self.super_experts = sorted(set(int(x) for x in (super_experts or [])))
        self._super_expert_set = set(self.super_experts)
        self.packed_expert_mask = [False for _ in range(len(self.experts))]
        if track_super_projected_weights:
            self.super_projected_weights: Dict[int, Dict[str, torch.Tensor]] = {}
        for key in self._SHARED_BASIS_BUFFER_KEYS:
            self.register_buffer(key, torch.empty(0, dtype=torch.float16), persistent=True)
        self._super_expert_items: List[Tuple[int, nn.Module]] = []
        self._super_weights: Optional[Tuple[torch.Tensor, torch.Tensor]] = None     # gate and up rows [E, 2I, H], down [E, H, I]
        self._super_global_to_local: Optional[torch.Tensor] = None
        self._super_map_of: Optional[tuple] = None          # (device, entries) of that map
        self._packed_expert_count = 0
        self._packed_intermediate_size = 0
        self._packed_global_to_local: Optional[torch.Tensor] = None
        self._packed_layer = None
        for tag in _TAGS:
            for f in _FIELDS:
                setattr(self, f"_{tag}_{f}_static", ())
        self._invalidate_runtime_cache()

    # ---- configuration ----------------------------------------------------------------------------
    def _runtime_device(self) -> torch.device:
        gate = getattr(self, "gate", None)
        weight = getattr(gate, "weight", None)
        if isinstance(weight, torch.Tensor):
            return weight.device
        return next(gate.parameters()).device

    def _set_buffer(self, name: str, tensor: torch.Tensor) -> None:
        setattr(self, name, tensor.detach().to(device=self._runtime_device(), dtype=torch.float16,
                                               non_blocking=True).contiguous())

    def set_shared_basis(self, gate_vh: torch.Tensor, up_vh: torch.Tensor, down_u: torch.Tensor) -> None:
        self._set_buffer("shared_vh_gate_proj", gate_vh)
        self._set_buffer("shared_vh_up_proj", up_vh)
        self._set_buffer("shared_u_down", down_u)
        self._invalidate_runtime_cache()

    def set_expert(self, expert_idx: int, expert_module: nn.Module, packed: bool) -> None:
        idx = int(expert_idx)
        self.experts[idx] = expert_module
        self.packed_expert_mask[idx] = bool(packed)
        self._invalidate_runtime_cache()

    def set_super_expert_projected_weights(self, expert_idx: int, gate_us: torch.Tensor, up_us: torch.Tensor,
                                           down_svh: torch.Tensor) -> None:
        if not hasattr(self, "super_projected_weights"):
            self.super_projected_weights = {}
        self.super_projected_weights[int(expert_idx)] = {
            "gate_us": gate_us.detach().to(dtype=torch.float16).contiguous(),
            "up_us": up_us.detach().to(dtype=torch.float16).contiguous(),
            "down_svh": down_svh.detach().to(dtype=torch.float16).contiguous(),
        }

    def _resize_basis_for(self, state_dict, prefix: str, assign: bool) -> None:
        for key in self._SHARED_BASIS_BUFFER_KEYS:
            t = state_dict.get(f"{prefix}{key}", None)
            if not isinstance(t, torch.Tensor):
                continue
            cur = getattr(self, key, None)
            if isinstance(cur, torch.Tensor) and cur.shape == t.shape and cur.dtype == t.dtype:
                continue
            setattr(self, key, t.detach() if assign else torch.empty_like(t))

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        self._resize_basis_for(state_dict, prefix, bool(local_metadata.get("assign_to_params_buffers", False)))
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        self._invalidate_runtime_cache()

    def _act_type(self) -> int:
        hidden_act = str(getattr(self.config, "hidden_act", "silu")).lower()
        if hidden_act != "silu":
            raise RuntimeError(f"Unsupported hidden_act for packed CUDA path: {hidden_act}")
        return 0

    # ---- runtime cache ----------------------------------------------------------------------------
    def _invalidate_runtime_cache(self) -> None:
        self._runtime_cache_ready = False
        self._runtime_cache_device: Optional[torch.device] = None
        self._runtime_warmed = False
        self._cached_token_count = -1
        self._cached_flat_token_ids: Optional[torch.Tensor] = None
        layer = getattr(self, "_packed_layer", None)
        if layer is not None:
            layer.close()
        self._packed_layer = None

    def _ensure_runtime_cache(self, device: torch.device) -> None:
        if self._runtime_cache_ready and self._runtime_cache_device == device:
            return
        super_items, packed_items = [], []
        for idx, module in enumerate(self.experts):
            if module is None:
                continue
            if idx in self._super_expert_set:
                super_items.append((idx, module))
            elif getattr(module, "is_bitsmoe_packed", False):
                packed_items.append((idx, module))
            else:
                raise RuntimeError(
                    f"Layer {self.layer_idx} expert {idx} is active but not packed. "
                    "BitsMoE forward expects non-super routed experts to use packed kernel.")
        self._super_expert_items = super_items
        self._packed_expert_count = len(packed_items)
        self._packed_intermediate_size = int(packed_items[0][1].intermediate_size) if packed_items else 0
        g2l = torch.full((self.num_experts,), -1, dtype=torch.int32)
        for local, (idx, _) in enumerate(packed_items):
            g2l[idx] = local
        self._packed_global_to_local = g2l.to(device)
        supers = torch.full((self.num_experts,), -1, dtype=torch.int32)
        for local, (idx, _) in enumerate(super_items):
            supers[idx] = local
        # map and stack outlive the cache where they still hold: a captured graph of the un-quantised experts reads them
        if not super_items:
            self._super_global_to_local = self._super_weights = None
        elif self._super_global_to_local is None or self._super_map_of != (device, supers.tolist()):
            self._super_global_to_local, self._super_map_of = supers.to(device), (device, supers.tolist())
        self._identity_map = self._packed_expert_count == self.num_experts and not super_items
        modules = [m for _, m in packed_items]
        for tag in _TAGS:
            for f in _FIELDS:
                setattr(self, f"_{tag}_{f}_static", tuple(getattr(m, f"{tag}_{f}_buffer") for m in modules))
        self._packed_layer = None
        if modules and device.type == "cuda" and _HAS_MLP_FORWARD_CUDA:
            from bitsmoe_b200.layer import PackedLayer
            self._act_type()
            self._packed_layer = PackedLayer.from_expert_modules(
                modules, self._packed_intermediate_size,
                int(self.shared_u_down.shape[1]) if self.shared_u_down.numel() else int(self.shared_vh_gate_proj.shape[0]),
                self.shared_vh_gate_proj, self.shared_vh_up_proj, self.shared_u_down, device=device)
        self._runtime_cache_ready = True
        self._runtime_cache_device = device
        self._runtime_warmed = False

    def _get_flat_token_ids(self, token_count: int, device: torch.device) -> torch.Tensor:
        ids = self._cached_flat_token_ids
        if ids is None or self._cached_token_count != token_count or ids.device != device:
            ids = torch.arange(token_count, dtype=torch.long, device=device).repeat_interleave(self.top_k)
            self._cached_flat_token_ids, self._cached_token_count = ids, token_count
        return ids

    # ---- routing / experts at the reference's internal boundaries -----------------------------------
    def _build_packed_routing(self, flat_selected_experts: torch.Tensor, flat_token_ids: torch.Tensor,
                              flat_route_weights_fp32: torch.Tensor):
        """-> (token_indices int32, expert_offsets int32 [E'+1], route_flat fp32) or None when the block has no
        packed experts.  Built by one kernel; the arrays keep their full length T*k and entries past
        expert_offsets[-1] are unspecified (the op walks expert_offsets)."""
        if self._packed_expert_count <= 0 or self._packed_global_to_local is None:
            return None
        from bitsmoe_b200.layer import route_build
        k = self.top_k
        tok, off, rw, _, _ = route_build(flat_selected_experts.reshape(-1, k), flat_route_weights_fp32.reshape(-1, k),
                                         self._packed_expert_count,
                                         None if self._identity_map else self._packed_global_to_local)
        return tok, off, rw

    def _run_super_experts(self, hidden_states, final_hidden_states, flat_selected_experts, flat_token_ids,
                           flat_route_weights_hidden) -> None:
        for expert_idx, module in self._super_expert_items:
            rows = (flat_selected_experts == expert_idx).nonzero(as_tuple=True)[0]
            if rows.numel() == 0:
                continue
            token_ids = flat_token_ids[rows]
            out = module(hidden_states.index_select(0, token_ids)) * flat_route_weights_hidden[rows].unsqueeze(-1)
            final_hidden_states.index_add_(0, token_ids, out.to(hidden_states.dtype))

    def _super_parts(self) -> Optional[List[List[torch.Tensor]]]:
        """[gate, up, down] weights of every un-quantised expert when all are bias-free SwiGLU MLPs of one shape and 16-bit type."""
        if str(getattr(self.config, "hidden_act", "silu")).lower() != "silu":
            return None
        parts = []
        for _, module in self._super_expert_items:
            if not runs_as_swiglu(module):
                return None
            w = [module._modules[n]._parameters.get("weight") for n in ("gate_proj", "up_proj", "down_proj")]
            if any(type(p) is not nn.Parameter for p in w):
                return None
            parts.append(w)
        g = parts[0][0]
        if g.dtype not in (torch.float16, torch.bfloat16):
            return None
        shape, dtype, device = g.shape, g.dtype, g.device
        back = shape[::-1]
        for gate, up, down in parts:
            if gate.shape != shape or up.shape != shape or down.shape != back:
                return None
            if gate.dtype != dtype or up.dtype != dtype or down.dtype != dtype or gate.device != device or up.device != device or down.device != device:
                return None
        return parts

    def _stacked_super_weights(self) -> Optional[Tuple[torch.Tensor, torch.Tensor]]:
        """The un-quantised experts' weights as two stacked tensors, whose slices the experts' own parameters become: nothing is held
        twice, and what is written to a parameter is what the kernels read.  Built again once a parameter lives somewhere else; whoever
        builds it waits for the device, as the packed part of the cache does."""
        parts = self._super_parts()
        if parts is None:
            return None
        if self._stack_holds(parts):
            return self._super_weights
        if not self._can_stack(parts):
            return None
        device = parts[0][0].device
        if device.type == "cuda":
            with torch.cuda.device(device):
                if torch.cuda.is_current_stream_capturing():
                    return None                  # the copies would run at the graph's replay
        with _stacking_lock(device):
            if not self._stack_holds(parts):     # else another thread has just built it
                inter, hidden = parts[0][0].shape
                with torch.inference_mode(False), torch.no_grad():    # the parameters stay ordinary tensors, whatever mode the first call is in
                    gu = parts[0][0].new_empty((len(parts), 2 * inter, hidden))
                    dn = parts[0][0].new_empty((len(parts), hidden, inter))
                    views = [(gu[i, :inter], gu[i, inter:], dn[i]) for i in range(len(parts))]
                    for w, vs in zip(parts, views):
                        for p, v in zip(w, vs):
                            v.copy_(p)
                    self._finish_copies(device)
                    for w, vs in zip(parts, views):
                        for p, v in zip(w, vs):
                            p.data = v
                self._super_weights = (gu, dn)
        return self._super_weights

    def _stack_holds(self, parts) -> bool:
        """Whether the experts' parameters are the slices of the stack."""
        if self._super_weights is None:
            return False
        gu, dn = self._super_weights
        inter, hidden = parts[0][0].shape
        if gu.shape != (len(parts), 2 * inter, hidden):
            return False
        # addresses, not views: this runs in every call
        size, at, down = inter * hidden * gu.element_size(), gu.data_ptr(), dn.data_ptr()
        for gate, up, dwn in parts:
            if gate.data_ptr() != at or up.data_ptr() != at + size or dwn.data_ptr() != down:
                return False
            if not (gate.is_contiguous() and up.is_contiguous() and dwn.is_contiguous()):
                return False
            at, down = at + 2 * size, down + size
        return True

    def _can_stack(self, parts) -> bool:
        """Whether every parameter has a storage of its own, or is a slice of this block's stack: moving one that others look into (an
        expert that several ids or blocks share, a view of a larger tensor) would part them, and move it back and forth."""
        held = () if self._super_weights is None else tuple(t.untyped_storage().data_ptr() for t in self._super_weights)
        flat = [p for w in parts for p in w]
        if len({p.data_ptr() for p in flat}) != len(flat):
            return False
        return all(p.untyped_storage().data_ptr() in held or p.untyped_storage().nbytes() == p.numel() * p.element_size() for p in flat)

    @staticmethod
    def _finish_copies(device: torch.device) -> None:
        """Calls on other streams use the slices as soon as they are the parameters, and the storage that the parameters leave goes back
        to the stream that it was made on: both have to wait until the copies are done, and what reads the old storage with them."""
        if device.type == "cuda":
            torch.cuda.synchronize(device)

    def _library_super_experts(self, x: torch.Tensor, topk_idx: torch.Tensor, topk_w: torch.Tensor,
                               residual: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
        """residual + the un-quantised experts' weighted outputs by the library (inference; no host sync, so a block with such experts
        can be captured into a CUDA graph), or None when the modules are of another kind."""
        if not x.is_cuda or torch.is_grad_enabled() or topk_idx.shape[-1] > 32:
            return None
        weights = self._stacked_super_weights()
        if weights is None or weights[0].dtype != x.dtype or weights[0].device != x.device:
            return None
        from bitsmoe_b200.layer import dense_experts
        return dense_experts(x, topk_idx, topk_w, *weights, global_to_local=self._super_global_to_local, residual=residual)

    def prepare_runtime_fastpath(self, warmup: bool = True) -> None:
        device = self._runtime_device()
        self._ensure_runtime_cache(device)
        if self._super_expert_items and device.type == "cuda":
            self._stacked_super_weights()
        if warmup:
            self._warmup_runtime_once(device)

    def _warmup_runtime_once(self, device: torch.device) -> None:
        if self._runtime_warmed or device.type != "cuda" or self._packed_layer is None:
            return
        if self.shared_vh_gate_proj.numel() == 0 or self.shared_vh_up_proj.numel() == 0:
            return
        x = torch.zeros((1, int(self.shared_vh_gate_proj.shape[1])), dtype=torch.float16, device=device)
        logits = torch.zeros((1, self.num_experts), dtype=torch.float32, device=device)
        with torch.no_grad():
            self._fused_forward(x, logits=logits)
        torch.cuda.synchronize(device)
        self._runtime_warmed = True

    def _packed_forward_cuda(self, h_gate_proj, h_up_proj, token_indices, expert_offsets_t, route_flat,
                             token_count: int) -> torch.Tensor:
        rank_out = int(self.shared_u_down.shape[1])
        if int(self._packed_intermediate_size) <= 0:
            raise RuntimeError(f"Layer {self.layer_idx} has no packed experts for CUDA path.")
        args = [getattr(self, f"_{tag}_{f}_static") for tag in _TAGS for f in _FIELDS]
        rank_accum = mlp_forward_cuda.moe_packed_forward(h_gate_proj, h_up_proj, token_indices, expert_offsets_t,
                                                         route_flat, *args, rank_out,
                                                         int(self._packed_intermediate_size), self._act_type())
        if rank_accum.shape[0] != token_count or rank_accum.shape[1] != rank_out:
            raise RuntimeError(f"Invalid rank_accum shape from CUDA kernel: got {tuple(rank_accum.shape)}, "
                               f"expected ({token_count}, {rank_out})")
        return torch.matmul(rank_accum.to(self.shared_u_down.dtype), self.shared_u_down.T)

    def _packed_forward_grouped(self, h_gate_proj, h_up_proj, token_indices, expert_offsets_t, route_flat,
                                token_count: int) -> torch.Tensor:
        if self.shared_u_down.numel() == 0:
            raise RuntimeError(f"Layer {self.layer_idx} missing shared_u_down for packed routed experts.")
        if not (_HAS_MLP_FORWARD_CUDA and mlp_forward_cuda is not None and h_gate_proj.is_cuda and h_up_proj.is_cuda):
            raise RuntimeError("Packed routed experts require CUDA mlp_forward extension; "
                               "python fallback is intentionally disabled.")
        return self._packed_forward_cuda(h_gate_proj, h_up_proj, token_indices, expert_offsets_t, route_flat, token_count)

    # ---- dense modules of the block on the library's kernels --------------------------------------------
    @staticmethod
    def _plain_linear(m) -> bool:
        return isinstance(m, nn.Linear) and m.bias is None

    def _library_gate_logits(self, x: torch.Tensor) -> Optional[torch.Tensor]:
        """x @ gate.weight.T by the library when the gate is a bias-free Linear on the GPU (inference), else None."""
        gate = getattr(self, "gate", None)
        if not (x.is_cuda and self._plain_linear(gate) and not torch.is_grad_enabled()):
            return None
        from bitsmoe_b200.layer import gate_logits
        return gate_logits(x, gate.weight)

    def _library_dense_mlp(self, x: torch.Tensor, mlp, token_gate=None) -> Optional[torch.Tensor]:
        """SwiGLU MLP ``mlp`` (gate_proj / up_proj / down_proj, bias-free, SiLU) by the library, scaled per token by
        sigmoid(token_gate(x)) when a one-output bias-free Linear is given; None when the module is of another kind."""
        parts = [getattr(mlp, n, None) for n in ("gate_proj", "up_proj", "down_proj")]
        if all(isinstance(p, Linear4) for p in parts):
            return self._library_dense_mlp4(x, parts, token_gate) if runs_as_swiglu(mlp) else None
        if not (x.is_cuda and all(self._plain_linear(p) for p in parts) and not torch.is_grad_enabled()):
            return None
        if token_gate is not None and not (self._plain_linear(token_gate) and token_gate.weight.shape[0] == 1):
            return None
        if parts[0].weight.shape[0] % 2:
            return None
        from bitsmoe_b200.layer import dense_mlp
        return dense_mlp(x, parts[0].weight, parts[1].weight, parts[2].weight,
                         None if token_gate is None else token_gate.weight)

    def _library_dense_mlp4(self, x: torch.Tensor, parts, token_gate) -> Optional[torch.Tensor]:
        """The same for an MLP whose Linears are held in 4 bits (``quantize_shared_experts``)."""
        if not (x.is_cuda and x.dtype in (torch.float16, torch.bfloat16) and not torch.is_grad_enabled()) or len({p.group_size for p in parts}) != 1:
            return None
        if token_gate is not None and not (self._plain_linear(token_gate) and token_gate.weight.shape[0] == 1):
            return None
        from bitsmoe_b200.layer import dense_mlp4
        return dense_mlp4(x, *(p.packed() for p in parts), group_size=parts[0].group_size,
                          token_gate_weight=None if token_gate is None else token_gate.weight.detach())

    def quantize_shared_experts(self, group_size: int = 128) -> int:
        """Holds the shared expert's three Linears in 4 bits from now on (one scale for every ``group_size`` columns of a row); returns
        how many were replaced.  For memory, a quarter of theirs, not for speed: a Qwen3-Next block then leaves its one-call path and takes 43 us
        instead of 33 for one token inside a graph, 88 instead of 72 for 64 (80 instead of 33 for one outside)."""
        n = 0
        for name in ("shared_expert", "shared_experts"):
            mlp = getattr(self, name, None)
            parts = [getattr(mlp, p, None) for p in ("gate_proj", "up_proj", "down_proj")]
            if not all(self._plain_linear(p) for p in parts):
                continue
            for p, lin in zip(("gate_proj", "up_proj", "down_proj"), parts):
                setattr(mlp, p, Linear4.from_linear(lin, group_size))
                n += 1
        return n

    def _bare_weight(self, module) -> Optional[torch.Tensor]:
        """The weight of a bias-free nn.Linear, else None (dict look-ups: this runs per layer and step)."""
        if not isinstance(module, nn.Linear) or module._parameters.get("bias") is not None:
            return None
        return module._parameters.get("weight")

    def _shared_weights(self):
        """(gate, up, down, token gate or None) weights of a shared expert the library can run, None when the block has
        no shared expert, False when it has one that only its own module can run."""
        return None

    def _one_call_forward(self, hidden_states: torch.Tensor):
        """Router, packed experts and shared expert in one library call -> (y in the input's shape, router logits), or
        None when a part of the block is not of the kind the library runs (the caller then goes through the stages)."""
        layer = self._packed_layer
        if layer is None or self._super_expert_items or not hidden_states.is_cuda or torch.is_grad_enabled():
            return None
        gate = self._bare_weight(self._modules.get("gate"))
        shared = self._shared_weights()
        if gate is None or shared is False:
            return None
        return layer.block_forward(hidden_states, gate, self.top_k, self.norm_topk_prob, hidden_states.dtype, shared,
                                   None if self._identity_map else self._packed_global_to_local)

    # ---- fused path -----------------------------------------------------------------------------------
    def _require_fused(self, x: torch.Tensor):
        if self.shared_vh_gate_proj.numel() == 0 or self.shared_vh_up_proj.numel() == 0:
            raise RuntimeError(f"Layer {self.layer_idx} missing shared_vh basis for packed routed experts.")
        if self.shared_u_down.numel() == 0:
            raise RuntimeError(f"Layer {self.layer_idx} missing shared_u_down for packed routed experts.")
        if self._packed_layer is None or not x.is_cuda:
            raise RuntimeError("Packed routed experts require CUDA mlp_forward extension; "
                               "python fallback is intentionally disabled.")
        return self._packed_layer

    def _fused_forward(self, x: torch.Tensor, logits: Optional[torch.Tensor] = None,
                       topk: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                       residual: Optional[torch.Tensor] = None, round_weights: bool = True) -> torch.Tensor:
        """x [T,H]; either router ``logits`` [T,E] (softmax/top-k run on the device) or a precomputed
        ``topk = (idx [T,k], weights [T,k])``.  Returns y [T,H] = packed experts (+ residual)."""
        layer = self._require_fused(x)
        g2l = None if self._identity_map else self._packed_global_to_local
        if topk is None:
            return layer.forward(x, logits, self.top_k, getattr(self, "norm_topk_prob", True),
                                 x.dtype if round_weights else None, residual=residual, global_to_local=g2l)
        from bitsmoe_b200.layer import route_build
        idx, w = topk
        tok, off, rw, _, _ = route_build(idx, w, self._packed_expert_count, g2l)
        hg, hu = layer.basis_project(x)
        acc = layer.experts_forward(hg, hu, tok, off, rw)
        return layer.combine_down_basis(acc, x.dtype, residual=residual)
