"""Low-rank adapters of many requests beside a projection that they share, on B200::

    y[r] = round( base[r] + scale[a] * B[a] (A[a] x[r]) )      a: the adapter of row r's request
    y[r] = round( base[r] )                                    for rows without one

``AdapterPlan`` sorts a batch's rows by adapter, once per step on the device; ``LowRankAdapters`` holds the adapters of one
projection (or of the experts of a MoE layer) and adds them to the projection's output in one launch for all requests.
``TernaryLinear(x, adapters=..., plan=...)`` and ``MoELayer(x, logits, adapters=..., plan=...)`` call them. Slots are loaded
and cleared in place, so captured graphs keep reading them. There is no CPU path.
"""

from __future__ import annotations

import ctypes

import torch

from .. import _lib
from ..kernels import ternary_b200 as kb

_UNAVAILABLE = "the B200 adapters are unavailable: {} not on a CUDA device and this backend has no CPU path"
_PADDED_RANKS = (16, 32, 64, 128)
_EXPERT_TILE = 16


def _int32(t: torch.Tensor, what: str) -> torch.Tensor:
    if not t.is_cuda:
        raise RuntimeError(_UNAVAILABLE.format(what + " are"))
    if t.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{what} must be int32 or int64")
    return t.contiguous() if t.dtype == torch.int32 else t.clamp(-1, 0x7fffffff).to(torch.int32).contiguous()


class AdapterPlan:
    """The rows of a batch sorted by adapter. ``slots`` [rows]: the adapter of each row, outside [0, n_adapters): none.

    ``rows`` [rows] int32: the row at each position (adapters in order, then the rows without one; a stable sort);
    ``offsets`` [n_adapters + 2] int32: where each adapter's positions start, then those without one, then the row count."""

    def __init__(self, slots: torch.Tensor, n_adapters: int):
        if slots.dim() != 1:
            raise RuntimeError("slots hold one adapter per row")
        self._build(None, slots, slots.size(0), n_adapters)

    @classmethod
    def from_requests(cls, offsets: torch.Tensor, slots: torch.Tensor, n_rows: int, n_adapters: int) -> "AdapterPlan":
        """The plan of a batch whose request i has rows ``offsets[i]`` .. ``offsets[i + 1]`` and adapter ``slots[i]``: offsets
        [R + 1], nondecreasing, slots [R], both on the device. Rows behind the last request (a padded batch) have none."""
        if offsets.dim() != 1 or slots.dim() != 1 or offsets.size(0) != slots.size(0) + 1:
            raise ValueError("offsets hold one entry per request + 1")
        self = cls.__new__(cls)
        self._build(offsets, slots, n_rows, n_adapters)
        return self

    def _build(self, offsets, slots, n_rows: int, n_adapters: int) -> None:
        lib = kb._require("auto")
        slots = _int32(slots, "slots")
        dev = slots.device
        if offsets is not None:
            offsets = _int32(offsets, "offsets")
            if offsets.device != dev:
                raise RuntimeError("offsets and slots must share one device")
        if n_adapters < 1 or n_adapters > 4095 or n_rows < 0:
            raise RuntimeError("a plan takes 1 to 4095 adapters")
        self.n_rows, self.n_adapters, self.device = n_rows, n_adapters, dev
        tile = self.tile = int(lib.dst_adapter_tile(n_rows))
        self.max_tiles = min(n_rows, -(-n_rows // tile) + n_adapters + 1)
        # one buffer: tiles, order, bins, offsets
        at_order = int(lib.dst_adapter_tile_capacity(n_rows, n_adapters + 1, tile))
        at_bins, at_offsets = at_order + n_rows, at_order + 2 * n_rows
        self._buf = torch.empty(at_offsets + n_adapters + 2, dtype=torch.int32, device=dev)
        self._at = at_order, at_bins, at_offsets
        base = self._buf.data_ptr()
        ws_bytes = int(lib.dst_adapter_plan_workspace_bytes(n_rows, n_adapters))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
        with kb._guard(dev):
            _lib.check(lib.dst_adapter_plan(offsets.data_ptr() if offsets is not None else None, slots.data_ptr(), slots.size(0), n_rows, n_adapters,
                                            tile, base + 4 * at_order, base + 4 * at_bins, base + 4 * at_offsets, base,
                                            ws.data_ptr() if ws is not None else None, ws_bytes, kb._stream(slots)))
        self._c = _lib.AdapterRowsC(rows=base + 4 * at_order, x_rows=base + 4 * at_order, tiles=base, max_tiles=self.max_tiles, tile=tile)
        self._ref = ctypes.byref(self._c)

    @property
    def rows(self) -> torch.Tensor:
        return self._buf[self._at[0]:self._at[1]]

    @property
    def offsets(self) -> torch.Tensor:
        return self._buf[self._at[2]:]

    def for_experts(self, ids: torch.Tensor, n_experts: int) -> "ExpertPlan":
        """The plan of the (token, choice) pairs of a MoE layer: ``ids`` [tokens, top_k] int32 or int64."""
        return ExpertPlan(self, ids, n_experts)


class ExpertPlan:
    """The (token, choice) pairs of a MoE layer sorted by expert and inside an expert by adapter. ``order`` [pairs] int64
    (token * top_k + choice at each position, -1 behind the last pair: ids outside [0, n_experts) are dropped) and ``offsets``
    [n_experts + 1] int64 take the place of ``sort_by_expert``'s results in the layer."""

    def __init__(self, plan: AdapterPlan, ids: torch.Tensor, n_experts: int):
        lib = kb._require("auto")
        if ids.dim() != 2 or ids.size(0) != plan.n_rows or ids.size(1) < 1:
            raise RuntimeError("ids are [tokens, top_k] of the plan's rows")
        if ids.is_cuda and ids.device != plan.device:
            raise RuntimeError("ids and the plan must share one device")
        ids = _int32(ids, "expert ids")
        T, k = ids.shape
        P, n, dev = T * k, plan.n_adapters, plan.device
        self.tokens, self.n_rows, self.n_adapters, self.n_experts, self.tile, self.device = T, P, n, n_experts, _EXPERT_TILE, dev
        self.max_tiles = min(P, -(-P // _EXPERT_TILE) + (n + 1) * n_experts)
        self.order = torch.empty(P, dtype=torch.int64, device=dev)
        self.offsets = torch.empty(n_experts + 1, dtype=torch.int64, device=dev)
        cap = int(lib.dst_adapter_tile_capacity(P, (n + 1) * n_experts, _EXPERT_TILE))
        self._buf = torch.empty(cap + P, dtype=torch.int32, device=dev)
        ws_bytes = int(lib.dst_adapter_plan_experts_workspace_bytes(P, n_experts))
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        base, src = self._buf.data_ptr(), plan._buf.data_ptr()
        with kb._guard(dev):
            _lib.check(lib.dst_adapter_plan_experts(ids.data_ptr(), T, k, n_experts, src + 4 * plan._at[0], src + 4 * plan._at[1], n, _EXPERT_TILE,
                                                    self.order.data_ptr(), self.offsets.data_ptr(), base + 4 * cap, base, ws.data_ptr(), ws_bytes,
                                                    kb._stream(ids)))
        self._pairs = _lib.AdapterRowsC(rows=None, x_rows=None, tiles=base, max_tiles=self.max_tiles, tile=_EXPERT_TILE)
        self._tokens = _lib.AdapterRowsC(rows=None, x_rows=base + 4 * cap, tiles=base, max_tiles=self.max_tiles, tile=_EXPERT_TILE)


class LowRankAdapters:
    """The adapters of one projection [N, K], or with ``experts`` of that projection of every expert of a MoE layer.

    ``rank``: the largest rank; a slot may hold a smaller one. ``parts`` 2: the projection's N rows are two stacked matrices
    with adapters of their own (gate and up, say). ``parts * rank`` is at most 128. Every slot starts empty: it adds nothing."""

    def __init__(self, n_adapters: int, K: int, N: int, rank: int, dtype=torch.bfloat16, experts: int | None = None, parts: int = 1, device="cuda"):
        if dtype not in (torch.bfloat16, torch.float16):
            raise RuntimeError("adapters are bf16 or fp16")
        if min(n_adapters, K, N, rank) < 1 or n_adapters > 4095 or (experts is not None and not 1 <= experts <= 4096):
            raise RuntimeError("invalid adapter sizes")
        if parts not in (1, 2) or N % parts != 0:
            raise RuntimeError("a projection has one part or two equal ones")
        self.rank_padded = next((p for p in _PADDED_RANKS if p >= rank and p * parts <= 128), None)
        if self.rank_padded is None:
            raise RuntimeError("parts * rank is at most 128")
        kb._require("auto")
        if torch.device(device).type != "cuda":
            raise RuntimeError(_UNAVAILABLE.format("the adapters are"))
        self.n_adapters, self.K, self.N, self.rank, self.dtype, self.experts, self.parts = n_adapters, K, N, rank, dtype, experts, parts
        E, Kp = experts or 1, -(-K // 32) * 32
        # A in steps of 32 values of K, the ranks of a step together: what a warp reads at once is one stretch of memory
        self._a = torch.zeros(n_adapters, E, Kp // 32, parts, self.rank_padded, 32, dtype=dtype, device=device)
        rows = n_adapters * E * N  # and 31 more, which the last step of columns may read
        self._b = torch.zeros(rows + 31, self.rank_padded, dtype=dtype, device=device)[:rows].view(n_adapters, E, N, self.rank_padded)
        self._scale = torch.zeros(n_adapters, dtype=torch.float32, device=device)
        self._ranks = torch.zeros(n_adapters, dtype=torch.int32, device=device)
        self.device = self._a.device
        self._c = _lib.AdaptersC(a=self._a.data_ptr(), b=self._b.data_ptr(), scale=self._scale.data_ptr(), ranks=self._ranks.data_ptr(),
                                 matrices_per_slot=E, K=K, K_padded=Kp, N=N, rank_padded=self.rank_padded, parts=parts, dtype=kb._ACT[dtype])
        self._ref = ctypes.byref(self._c)

    def load(self, slot: int, A: torch.Tensor, B: torch.Tensor, scale: float = 1.0) -> None:
        """Put an adapter into ``slot``: A [parts * r, K], B [N, r] (with ``experts``: [experts, ...] each), r <= ``rank``."""
        if not 0 <= slot < self.n_adapters:
            raise IndexError(f"slot {slot} of {self.n_adapters}")
        lead = () if self.experts is None else (self.experts,)
        r = B.size(-1)
        if tuple(A.shape) != (*lead, self.parts * r, self.K) or tuple(B.shape) != (*lead, self.N, r) or not 1 <= r <= self.rank:
            raise RuntimeError("inconsistent adapter shapes")
        self.clear(slot)
        wide = torch.zeros(A.numel() // (self.parts * r * self.K), self.parts, r, self._a.size(2) * 32, dtype=self.dtype, device=self.device)
        wide[..., :self.K] = A.reshape(-1, self.parts, r, self.K)
        self._a[slot, ..., :r, :] = wide.unflatten(-1, (-1, 32)).permute(0, 3, 1, 2, 4)
        self._b[slot, ..., :r] = B.reshape(-1, self.N, r)
        self._scale[slot] = scale
        self._ranks[slot] = r

    def clear(self, slot: int) -> None:
        """Empty a slot: its requests get the projection alone."""
        if not 0 <= slot < self.n_adapters:
            raise IndexError(f"slot {slot} of {self.n_adapters}")
        self._a[slot].zero_()
        self._b[slot].zero_()
        self._ranks[slot] = 0

    def __call__(self, x: torch.Tensor, plan, base: torch.Tensor | None = None, out_dtype=None, out: torch.Tensor | None = None,
                 pair_rows: bool = False) -> torch.Tensor:
        """x [rows, K] and the projection's output ``base`` [rows, N] (float32, bf16 or fp16; None: zeros) -> [rows, N] of
        ``out_dtype`` (default: the base's type, without one x's), into ``out`` if given, which may be ``base`` itself.

        With ``experts`` the plan is an ``ExpertPlan``, base and result hold one row per pair in its order, x one per token
        (``pair_rows``: one per pair too). Positions behind its last pair are not written."""
        if not x.is_cuda:
            raise RuntimeError(_UNAVAILABLE.format("activations are"))
        pairs = isinstance(plan, ExpertPlan)
        if pairs != (self.experts is not None) or plan.n_adapters != self.n_adapters or (pairs and plan.n_experts != self.experts):
            raise RuntimeError("the plan was made for other adapters")
        if pair_rows and not pairs:
            raise RuntimeError("pair_rows goes with an expert plan")
        if x.dtype != self.dtype:
            raise TypeError(f"the adapters take {self.dtype} activations")
        P = plan.n_rows
        if x.dim() != 2 or x.size(1) != self.K or x.size(0) != (plan.tokens if pairs and not pair_rows else P):
            raise RuntimeError("inconsistent adapter shapes")
        x = _rows(x)
        if base is not None:
            if base.dim() != 2 or tuple(base.shape) != (P, self.N) or base.dtype not in kb._OUT:
                raise RuntimeError("the base is float32, bf16 or fp16 [rows, N]")
            base = _rows(base)
        if out is None:
            out = torch.empty(P, self.N, dtype=out_dtype or (base.dtype if base is not None else x.dtype), device=x.device)
        if out.dim() != 2 or tuple(out.shape) != (P, self.N) or out.dtype not in kb._OUT or (out_dtype is not None and out.dtype != out_dtype) \
                or (P > 0 and out.stride(1) != 1) or (P > 1 and out.stride(0) < self.N):
            raise RuntimeError("the result is float32, bf16 or fp16 [rows, N]")
        if not (self.device == plan.device == x.device == out.device) or (base is not None and base.device != x.device):
            raise RuntimeError("adapters, plan and tensors must share one device")
        if P == 0:
            return out
        c = plan._ref if not pairs else ctypes.byref(plan._pairs if pair_rows else plan._tokens)
        with kb._guard(x.device):
            _lib.check(kb._require("auto").dst_adapter_apply(
                self._ref, c, x.data_ptr(), max(x.stride(0), self.K), base.data_ptr() if base is not None else None,
                kb._OUT[base.dtype] if base is not None else 0, max(base.stride(0), self.N) if base is not None else self.N,
                out.data_ptr(), kb._OUT[out.dtype], max(out.stride(0), self.N), kb._stream(x)))
        return out


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Rows of neighbouring elements, one behind the other at any distance; anything else is copied."""
    return t if t.stride(1) == 1 and (t.stride(0) >= t.size(1) or t.size(0) == 1) else t.contiguous()
