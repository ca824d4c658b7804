"""PyTorch-facing wrappers of libfns_hip.so (device memory and streams come from torch; the compute is the HIP
library's). Names, argument meaning and error behaviour follow the reference's kernel-launch API
(reference include/fns/ggml_kernels.h, src/kernels.cuh): a bad type or shape raises FnsError where the reference
aborts. All tensors are CUDA (HIP) tensors; launches go on torch's current stream.
"""
from __future__ import annotations

import ctypes

import numpy as np
import torch

from ._lib import call, lib

Q8_0, Q8_1, Q3_K, Q4_K, Q5_K, Q6_K = 8, 9, 11, 12, 13, 14
IQ3_XXS, IQ3_S, IQ2_S, IQ4_XS = 18, 21, 22, 23
F32, F16, BF16 = 0, 1, 30
GATING_SOFTMAX, GATING_SIGMOID = 0, 1
ROPE_NONE, ROPE_HALVES, ROPE_PAIRS = 0, 1, 2
STATUS_EXCHANGE_TIMEOUT = 1  # FNS_STATUS_EXCHANGE_TIMEOUT
# bytes per 256 values of a row (a K-quant block; 8 Q8_0 blocks)
BLOCK_BYTES = {Q8_0: 272, Q3_K: 110, Q4_K: 144, Q5_K: 176, Q6_K: 210, IQ3_XXS: 98, IQ3_S: 110, IQ2_S: 82, IQ4_XS: 136}
TYPE_NAMES = {Q8_0: "Q8_0", Q3_K: "Q3_K", Q4_K: "Q4_K", Q5_K: "Q5_K", Q6_K: "Q6_K", IQ3_XXS: "IQ3_XXS",
              IQ3_S: "IQ3_S", IQ2_S: "IQ2_S", IQ4_XS: "IQ4_XS"}


def _status_dst(t: torch.Tensor):
    """Pointer of a status collect's destination: a device tensor or pinned host memory of at least 4 bytes."""
    if t.numel() * t.element_size() < 4 or not (t.is_cuda or t.is_pinned()):
        raise ValueError("status destination: a device or pinned host tensor of at least 4 bytes")
    return ctypes.c_void_p(t.data_ptr())


def _p(t: torch.Tensor | None):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("expected a device tensor")
    return ctypes.c_void_p(t.data_ptr())


def _s():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def row_bytes(qtype: int, ncols: int) -> int:
    return BLOCK_BYTES[qtype] * (ncols // 256)


def q8_1_row_bytes(ncols: int) -> int:
    return int(lib().fns_hip_q8_1_row_bytes(ncols))


def _empty_f32(*shape, like: torch.Tensor) -> torch.Tensor:
    return torch.empty(*shape, dtype=torch.float32, device=like.device)


def quantize_q8_1(x: torch.Tensor, xq: torch.Tensor | None = None) -> torch.Tensor:
    x = x.contiguous()
    ncols = x.shape[-1]
    nrows = x.numel() // ncols
    if xq is None:
        xq = torch.zeros(nrows, q8_1_row_bytes(ncols), dtype=torch.uint8, device=x.device)
    call("fns_hip_quantize_q8_1", _p(x), _p(xq), ncols, nrows, _s())
    return xq


def mmvq(qtype: int, w: torch.Tensor, ncols: int, nrows: int, xq: torch.Tensor, n_cols: int,
         dst: torch.Tensor | None = None) -> torch.Tensor:
    dst = _empty_f32(n_cols, nrows, like=xq) if dst is None else dst
    call("fns_hip_mmvq", qtype, _p(w), ncols, nrows, _p(xq), _p(dst), n_cols, _s())
    return dst


def mmvq_ids(qtype: int, w: torch.Tensor, ncols: int, nrows: int, n_mats: int, xq: torch.Tensor, n_xq: int,
             ids: torch.Tensor, dst: torch.Tensor | None = None) -> torch.Tensor:
    n_ids = ids.numel()
    dst = _empty_f32(n_ids, nrows, like=xq) if dst is None else dst
    call("fns_hip_mmvq_ids", qtype, _p(w), ncols, nrows, n_mats, _p(xq), n_xq, _p(ids), n_ids, _p(dst), _s())
    return dst


def mmvq_swiglu(qtype: int, w_gate: torch.Tensor, w_up: torch.Tensor, ncols: int, nrows: int, xq: torch.Tensor,
                dst: torch.Tensor | None = None) -> torch.Tensor:
    dst = _empty_f32(nrows, like=xq) if dst is None else dst
    call("fns_hip_mmvq_swiglu", qtype, _p(w_gate), _p(w_up), ncols, nrows, _p(xq), _p(dst), _s())
    return dst


def mmvq_ids_swiglu_shared(qtype: int, w_gate: torch.Tensor, w_up: torch.Tensor, ncols: int, nrows: int, n_mats: int,
                           xq: torch.Tensor, ids: torch.Tensor, sh_gate: torch.Tensor | None = None,
                           sh_up: torch.Tensor | None = None, dst: torch.Tensor | None = None,
                           sh_dst: torch.Tensor | None = None):
    n_ids = ids.numel()
    dst = _empty_f32(n_ids, nrows, like=xq) if dst is None else dst
    if sh_gate is not None and sh_dst is None:
        sh_dst = _empty_f32(nrows, like=xq)
    call("fns_hip_mmvq_ids_swiglu_shared", qtype, _p(w_gate), _p(w_up), ncols, nrows, n_mats, _p(xq), _p(ids), n_ids,
         _p(dst), _p(sh_gate), _p(sh_up), _p(sh_dst), _s())
    return dst, sh_dst


def mmvq_experts_swiglu(qtype: int, table: torch.Tensor, gate_off: int, up_off: int, ncols: int, nrows: int,
                        xq: torch.Tensor, n_xq: int, ids: torch.Tensor, dst: torch.Tensor | None = None):
    n_ids = ids.numel()
    dst = _empty_f32(n_ids, nrows, like=xq) if dst is None else dst
    call("fns_hip_mmvq_experts_swiglu", qtype, _p(table), gate_off, up_off, ncols, nrows, _p(xq), n_xq, _p(ids),
         n_ids, _p(dst), _s())
    return dst


def mmvq_experts(qtype: int, table: torch.Tensor, off: int, ncols: int, nrows: int, xq: torch.Tensor, n_xq: int,
                 ids: torch.Tensor, dst: torch.Tensor | None = None):
    n_ids = ids.numel()
    dst = _empty_f32(n_ids, nrows, like=xq) if dst is None else dst
    call("fns_hip_mmvq_experts", qtype, _p(table), off, ncols, nrows, _p(xq), n_xq, _p(ids), n_ids, _p(dst), _s())
    return dst


def mmvq_supports(qtype: int) -> bool:
    return bool(lib().fns_hip_mmvq_supports(qtype))


def rms_norm_q8_1(x: torch.Tensor, w: torch.Tensor, eps: float):
    x = x.contiguous()
    n = x.shape[-1]
    rows = x.numel() // n
    out = torch.empty_like(x)
    xq = torch.zeros(rows, q8_1_row_bytes(n), dtype=torch.uint8, device=x.device)
    call("fns_hip_rms_norm_q8_1", _p(x), _p(w), _p(out), _p(xq), n, ctypes.c_float(eps), rows, _s())
    return out, xq


def _dtype_code(w: torch.Tensor) -> int:
    if w.dtype == torch.float32:
        return F32
    if w.dtype == torch.bfloat16:
        return BF16
    raise ValueError(f"router dtype {w.dtype} not supported")


def gemv_router(w: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    nrows, ncols = w.shape
    x = x.contiguous().view(-1, ncols)
    y = _empty_f32(x.shape[0], nrows, like=x)
    call("fns_hip_gemv_router", _dtype_code(w), _p(w), _p(x), _p(y), ncols, nrows, x.shape[0], _s())
    return y


def gemm_router(w: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    nrows, ncols = w.shape
    x = x.contiguous().view(-1, ncols)
    y = _empty_f32(x.shape[0], nrows, like=x)
    call("fns_hip_gemm_router", _dtype_code(w), _p(w), _p(x), _p(y), ncols, nrows, x.shape[0], _s())
    return y


def route_topk(logits: torch.Tensor, k: int, gating: int = GATING_SOFTMAX, norm: bool = True):
    logits = logits.contiguous()
    n_expert = logits.shape[-1]
    n_tok = logits.numel() // n_expert
    ids = torch.empty(n_tok, k, dtype=torch.int32, device=logits.device)
    w = _empty_f32(n_tok, k, like=logits)
    call("fns_hip_route_topk", _p(logits), _p(ids), _p(w), n_expert, k, n_tok, gating, int(norm), _s())
    return ids, w


def count_routes(ids: torch.Tensor, counts: torch.Tensor) -> None:
    call("fns_hip_count_routes", _p(ids), _p(counts), ids.numel(), _s())


def swiglu(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    n = g.shape[-1]
    act = torch.empty_like(g)
    call("fns_hip_swiglu", _p(g.contiguous()), _p(u.contiguous()), _p(act), n, g.numel() // n, _s())
    return act


def glu_mmvq(g: torch.Tensor, u: torch.Tensor) -> torch.Tensor:
    act = torch.empty_like(g)
    call("fns_hip_glu_mmvq", _p(g.contiguous()), _p(u.contiguous()), _p(act), g.numel(), _s())
    return act


def amax_guard(act: torch.Tensor) -> torch.Tensor:
    """In place: act[r] /= e_r; returns escale [rows]."""
    n = act.shape[-1]
    rows = act.numel() // n
    escale = _empty_f32(rows, like=act)
    call("fns_hip_amax_guard", _p(act), _p(escale), n, rows, _s())
    return escale


def amax_guard_q8_1(act: torch.Tensor):
    n = act.shape[-1]
    rows = act.numel() // n
    escale = _empty_f32(rows, like=act)
    xq = torch.zeros(rows, q8_1_row_bytes(n), dtype=torch.uint8, device=act.device)
    call("fns_hip_amax_guard_q8_1", _p(act.contiguous()), _p(escale), _p(xq), n, rows, _s())
    return escale, xq


def moe_combine(dexp: torch.Tensor, w: torch.Tensor, escale=None, sh=None, x=None, out=None) -> torch.Tensor:
    """dexp [T][k][n], w [T][k] -> out [T][n] = (sum_j (dexp_j * e_j) * w_j + sh) + x."""
    T, k, n = dexp.shape
    out = _empty_f32(T, n, like=dexp) if out is None else out
    call("fns_hip_moe_combine", _p(dexp.contiguous()), _p(escale), _p(w.contiguous()), _p(sh), _p(x), _p(out), n, k,
         T, _s())
    return out


class ExpertSlots:
    """Fully resident expert storage: expert e is one slot [gate | up | down] of raw GGUF blocks at
    base + e * slot_bytes (256-byte aligned), plus a device table of slot pointers - the reference engine's
    `exp_table` / `gate_bytes` / `up_bytes` contract (reference include/fns/engine.h:28-32, src/engine.cu:375-471),
    in the trivial case where every expert lives in HBM. `pad` bytes of zeros follow the last slot
    (reference src/engine.cu:42-45).
    """

    def __init__(self, n_expert: int, gate_bytes: int, up_bytes: int, down_bytes: int, pad: int = 4096):
        self.n_expert = n_expert
        self.gate_bytes, self.up_bytes, self.down_bytes = gate_bytes, up_bytes, down_bytes
        raw = gate_bytes + up_bytes + down_bytes
        self.slot_bytes = (raw + 255) // 256 * 256
        self.gate_off, self.up_off, self.down_off = 0, gate_bytes, gate_bytes + up_bytes
        self.storage = torch.zeros(n_expert * self.slot_bytes + pad, dtype=torch.uint8, device="cuda")
        base = self.storage.data_ptr()
        self.table = torch.tensor([base + e * self.slot_bytes for e in range(n_expert)], dtype=torch.int64,
                                  device="cuda")

    @classmethod
    def from_tensors(cls, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, pad: int = 4096):
        """gate/up/down: uint8 [n_expert][bytes of one expert matrix] (host or device)."""
        s = cls(gate.shape[0], gate.shape[1], up.shape[1], down.shape[1], pad)
        for name, t in (("gate", gate), ("up", up), ("down", down)):
            s.view(name).copy_(t.to("cuda"))
        return s

    def view(self, name: str) -> torch.Tensor:
        """[n_expert][bytes] strided view of one matrix kind inside the slots."""
        off = {"gate": self.gate_off, "up": self.up_off, "down": self.down_off}[name]
        size = {"gate": self.gate_bytes, "up": self.up_bytes, "down": self.down_bytes}[name]
        slots = self.storage[: self.n_expert * self.slot_bytes].view(self.n_expert, self.slot_bytes)
        return slots[:, off: off + size]

    def expert_bytes(self, e: int) -> torch.Tensor:
        return self.storage[e * self.slot_bytes: (e + 1) * self.slot_bytes]


class MoeLayerDesc(ctypes.Structure):
    """Mirror of FnsMoeLayer (include/fns_hip.h)."""
    _fields_ = [
        ("hidden", ctypes.c_int), ("inter", ctypes.c_int), ("n_expert", ctypes.c_int), ("k", ctypes.c_int),
        ("gating", ctypes.c_int), ("norm_w", ctypes.c_int), ("guard", ctypes.c_int),
        ("router_dtype", ctypes.c_int), ("router_w", ctypes.c_void_p),
        ("gu_type", ctypes.c_int), ("down_type", ctypes.c_int),
        ("table", ctypes.c_void_p), ("gate_off", ctypes.c_size_t), ("up_off", ctypes.c_size_t),
        ("down_off", ctypes.c_size_t), ("router_bias", ctypes.c_void_p),
        ("ffn_norm", ctypes.c_void_p), ("norm_eps", ctypes.c_float), ("shexp_inter", ctypes.c_int),
        ("shexp_gu_type", ctypes.c_int), ("shexp_down_type", ctypes.c_int),
        ("shexp_gate", ctypes.c_void_p), ("shexp_up", ctypes.c_void_p), ("shexp_down", ctypes.c_void_p),
        ("prefetch", ctypes.c_void_p), ("prefetch_bytes", ctypes.c_size_t),
    ]


WS_SECTIONS = ("logits", "xq", "ids", "w", "act", "escale")

PATH_AUTO, PATH_THREE_KERNELS = 0, 1


class decode_path:
    """Context manager (test hook fns_hip_moe_set_path): restricts the decode path of the calls inside it."""

    def __init__(self, path: int):
        self.path = path

    def __enter__(self):
        call("fns_hip_moe_set_path", self.path)
        return self

    def __exit__(self, *exc):
        call("fns_hip_moe_set_path", PATH_AUTO)
        return False


class MoeLayer:
    """One MoE FFN layer resident in HBM: fp32/bf16 router + expert slots, run by fns_hip_moe_layer."""

    def __init__(self, router_w: torch.Tensor, slots: ExpertSlots, gu_type: int, down_type: int, hidden: int,
                 inter: int, k: int, gating: int = GATING_SOFTMAX, norm: bool = True, guard: bool = False,
                 router_bias: torch.Tensor | None = None, ffn_norm: torch.Tensor | None = None,
                 norm_eps: float = 1e-6, shexp: dict | None = None):
        """shexp: the shared expert, {"gate", "up", "down": uint8 block tensors, "inter": width, "gu_type",
        "down_type"} (the reference's gate_shexp / up_shexp / down_shexp); ffn_norm: f32 [hidden] RMSNorm weights."""
        self.router_w, self.slots, self.router_bias = router_w, slots, router_bias
        self.ffn_norm, self.shexp = ffn_norm, shexp
        sh = shexp or {}
        self.desc = MoeLayerDesc(hidden, inter, slots.n_expert, k, gating, int(norm), int(guard),
                                 _dtype_code(router_w), router_w.data_ptr(), gu_type, down_type,
                                 slots.table.data_ptr(), slots.gate_off, slots.up_off, slots.down_off,
                                 router_bias.data_ptr() if router_bias is not None else None,
                                 ffn_norm.data_ptr() if ffn_norm is not None else None, norm_eps,
                                 sh.get("inter", 0), sh.get("gu_type", 0), sh.get("down_type", 0),
                                 sh["gate"].data_ptr() if sh else None, sh["up"].data_ptr() if sh else None,
                                 sh["down"].data_ptr() if sh else None)

    @classmethod
    def from_gguf(cls, file: "GgufFile", layer: int) -> "MoeLayer":
        """MoE layer `layer` of a GGUF checkpoint made resident in HBM by fns_hip_moe_layer_from_gguf (expert slots,
        table, router, norm and shared expert in library-owned device memory, freed with this object)."""
        obj = cls.__new__(cls)
        obj.desc = MoeLayerDesc()
        obj.router_w = obj.slots = obj.router_bias = obj.ffn_norm = obj.shexp = None
        obj._file = file  # the metadata stays readable while the layer lives
        res = ctypes.c_void_p()
        call("fns_hip_moe_layer_from_gguf", file.handle, layer, ctypes.byref(res), ctypes.byref(obj.desc))
        obj._resident = res
        return obj

    def __del__(self):
        res = getattr(self, "_resident", None)
        if res:
            lib().fns_hip_moe_resident_free(res)
            self._resident = None

    def workspace_layout(self, n_tok: int):
        offs = (ctypes.c_size_t * 6)()
        total = ctypes.c_size_t()
        call("fns_hip_moe_workspace_layout", ctypes.byref(self.desc), n_tok, offs, ctypes.byref(total))
        return list(offs), total.value

    def workspace(self, n_tok: int) -> torch.Tensor:
        _, total = self.workspace_layout(n_tok)
        return torch.zeros(total, dtype=torch.uint8, device="cuda")

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None, ws: torch.Tensor | None = None,
                 x_resid: torch.Tensor | None = None) -> torch.Tensor:
        x = x.contiguous()
        n_tok = x.numel() // self.desc.hidden
        out = torch.empty_like(x) if out is None else out
        ws = self.workspace(n_tok) if ws is None else ws
        call("fns_hip_moe_layer", ctypes.byref(self.desc), _p(x), _p(x_resid), _p(out), n_tok, _p(ws), ws.numel(), _s())
        return out

    def status(self, ws: torch.Tensor | None, n_tok: int = 1, clear: bool = False) -> int:
        """The workspace's sticky status word (FNS_STATUS_* bits; 0: every call so far completed its exchange)."""
        st = ctypes.c_uint32()
        call("fns_hip_moe_layer_status", ctypes.byref(self.desc), n_tok, _p(ws), int(clear), ctypes.byref(st), _s())
        return st.value

    def status_collect(self, ws: torch.Tensor | None, dst: torch.Tensor, n_tok: int = 1) -> None:
        """Enqueues the graph-capturable collect (fns_hip_moe_layer_status_collect): a non-zero status word is ORed
        into dst[0] (a uint32-sized tensor, device or pinned host) and cleared."""
        call("fns_hip_moe_layer_status_collect", ctypes.byref(self.desc), n_tok, _p(ws), _status_dst(dst), _s())

    def kernels(self, n_tok: int = 1) -> int:
        """Kernels one call at n_tok tokens launches on the current device: 2 (router + fused layer) or 3 (router,
        gate/up, down)."""
        k = ctypes.c_int()
        call("fns_hip_moe_layer_kernels", ctypes.byref(self.desc), n_tok, ctypes.byref(k))
        return k.value

    def stage(self, stage: int, x: torch.Tensor, out: torch.Tensor, ws: torch.Tensor,
              x_resid: torch.Tensor | None = None) -> None:
        """Launch one of the layer's three kernels (0 router, 1 gate/up, 2 down + combine)."""
        n_tok = x.numel() // self.desc.hidden
        call("fns_hip_moe_layer_stage", ctypes.byref(self.desc), stage, _p(x), _p(x_resid), _p(out), n_tok, _p(ws),
             ws.numel(), _s())

    def profiled(self, x: torch.Tensor, out: torch.Tensor, ws: torch.Tensor, events) -> None:
        """Full layer with torch.cuda.Event markers before each kernel and after the last (4 events, recorded)."""
        n_tok = x.numel() // self.desc.hidden
        arr = (ctypes.c_void_p * 4)(*[e.cuda_event for e in events])
        call("fns_hip_moe_layer_profiled", ctypes.byref(self.desc), _p(x), None, _p(out), n_tok, _p(ws), ws.numel(),
             arr, _s())

    def trace(self, ws: torch.Tensor, n_tok: int) -> dict:
        """Views of the intermediates a call left in its workspace."""
        offs, _ = self.workspace_layout(n_tok)
        d = self.desc
        sizes = {"logits": (torch.float32, (n_tok, d.n_expert)), "xq": (torch.uint8, (n_tok, q8_1_row_bytes(d.hidden))),
                 "ids": (torch.int32, (n_tok, d.k)), "w": (torch.float32, (n_tok, d.k)),
                 "act": (torch.float32, (n_tok * d.k, d.inter)), "escale": (torch.float32, (n_tok * d.k,))}
        out = {}
        for name, off in zip(WS_SECTIONS, offs):
            dt, shape = sizes[name]
            n = int(np.prod(shape)) * torch.tensor([], dtype=dt).element_size()
            out[name] = ws[off:off + n].view(dt).view(*shape)
        return out


PREFILL_SECTIONS = ("logits", "ids", "w", "xpack", "apack", "dexp")


def _split_of_i8(rows: torch.Tensor, ncols: int) -> torch.Tensor:
    """The split image rows (uint8 [n][ncols / 256 * 1056]: every code times its scale as two f16 halves, then the sums)
    that int8 image rows (per 256 columns 320 bytes: int8 codes, 8 f32 block scales, 32 bytes of scaled sums) define: the
    same codes, scales and sums."""
    n, nb = rows.shape[0], ncols // 256
    sb = rows[:, : nb * 320].contiguous().view(n, nb, 320)
    q = sb[:, :, :256].contiguous().view(torch.int8).float().view(n, nb, 8, 32)
    x = q * sb[:, :, 256:288].contiguous().view(torch.float32).unsqueeze(3)  # exact in f32
    x = x.view(n, nb, 32, 8)[..., [0, 2, 1, 3, 4, 6, 5, 7]].reshape(n, nb, 2, 128)
    hi = x.half()
    main = torch.cat([hi, (x - hi.float()).half()], 3).reshape(n, nb * 512).view(torch.uint8)
    return torch.cat([main, sb[:, :, 288:].reshape(n, nb * 32)], 1)


class MoePrefill:
    """Prefill (batched) form of a MoeLayer: fns_hip_moe_prefill over n_tok tokens."""

    def __init__(self, layer: MoeLayer):
        self.layer = layer

    def workspace_layout(self, n_tok: int):
        offs = (ctypes.c_size_t * 6)()
        total = ctypes.c_size_t()
        call("fns_hip_moe_prefill_workspace", ctypes.byref(self.layer.desc), n_tok, offs, ctypes.byref(total))
        return list(offs), total.value

    def workspace(self, n_tok: int) -> torch.Tensor:
        return torch.zeros(self.workspace_layout(n_tok)[1], dtype=torch.uint8, device="cuda")

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None, ws: torch.Tensor | None = None,
                 x_resid: torch.Tensor | None = None) -> torch.Tensor:
        x = x.contiguous()
        n_tok = x.numel() // self.layer.desc.hidden
        out = torch.empty_like(x) if out is None else out
        ws = self.workspace(n_tok) if ws is None else ws
        call("fns_hip_moe_prefill", ctypes.byref(self.layer.desc), _p(x), _p(x_resid), _p(out), n_tok, _p(ws),
             ws.numel(), _s())
        return out

    def status(self, ws: torch.Tensor, n_tok: int, clear: bool = False) -> int:
        """The workspace's sticky status word (FNS_STATUS_* bits; 0: every fused gate/up + down wait so far completed)."""
        st = ctypes.c_uint32()
        call("fns_hip_moe_prefill_status", ctypes.byref(self.layer.desc), n_tok, _p(ws), int(clear), ctypes.byref(st),
             _s())
        return st.value

    def status_collect(self, ws: torch.Tensor, dst: torch.Tensor, n_tok: int) -> None:
        """Enqueues the graph-capturable collect (fns_hip_moe_prefill_status_collect) into dst[0]."""
        call("fns_hip_moe_prefill_status_collect", ctypes.byref(self.layer.desc), n_tok, _p(ws), _status_dst(dst),
             _s())

    def section(self, n_tok: int, index: int) -> tuple[int, int]:
        """(byte offset, bytes) of workspace section `index` (fns_hip_moe_prefill_section)."""
        off, size = ctypes.c_size_t(), ctypes.c_size_t()
        call("fns_hip_moe_prefill_section", ctypes.byref(self.layer.desc), n_tok, index, ctypes.byref(off),
             ctypes.byref(size))
        return off.value, size.value

    def trace(self, ws: torch.Tensor, n_tok: int) -> dict:
        """The intermediates a call left in its workspace: views of logits, ids, w and dexp, the activation images of x
        in the split form ("xpack", [n_tok][split row bytes]) and of act ("apack", [n_tok * k][split row bytes], by (token, slot)), the guard
        scales ("escale") and, with the F16 guard, the f32 act rows after the division ("act")."""
        d = self.layer.desc
        P = n_tok * d.k
        spec = {"logits": (0, torch.float32, (n_tok, d.n_expert)), "ids": (1, torch.int32, (n_tok, d.k)),
                "w": (2, torch.float32, (n_tok, d.k)), "xpack": (3, torch.uint8, (n_tok, -1)),
                "apack": (4, torch.uint8, (P, -1)), "dexp": (5, torch.float32, (n_tok, d.k, d.hidden)),
                "act": (9, torch.float32, (P, d.inter)), "escale": (10, torch.float32, (P,))}
        out = {}
        for name, (idx, dt, shape) in spec.items():
            off, n = self.section(n_tok, idx)
            if n:
                out[name] = ws[off: off + n].view(dt).view(*shape)
        form, stride = ctypes.c_int(), ctypes.c_size_t()
        for name, idx, ncols in (("xpack", 3, d.hidden), ("apack", 4, d.inter)):
            call("fns_hip_moe_prefill_image", ctypes.byref(d), idx, ctypes.byref(form), ctypes.byref(stride))
            n = out[name].shape[0]
            rows = out[name].reshape(-1)[: n * stride.value].view(n, stride.value)
            out[name] = _split_of_i8(rows, ncols) if form.value else rows[:, : ncols // 256 * 1056]
        return out


def mmq_q8_1_bytes(ncols: int, nrows: int) -> int:
    return int(lib().fns_hip_mmq_q8_1_bytes(ncols, nrows))


def mmq(qtype: int, w: torch.Tensor, ncols: int, nrows: int, x: torch.Tensor, xq: torch.Tensor | None = None,
        out: torch.Tensor | None = None) -> torch.Tensor:
    """dst [n_tok][nrows] = W . q8_1(x); xq: scratch of mmq_q8_1_bytes(ncols, n_tok) bytes (allocated if None)."""
    x = x.contiguous()
    n_tok = x.numel() // ncols
    if xq is None:
        xq = torch.zeros(mmq_q8_1_bytes(ncols, n_tok), dtype=torch.uint8, device=x.device)
    dst = _empty_f32(n_tok, nrows, like=x) if out is None else out
    call("fns_hip_mmq", qtype, _p(w), ncols, nrows, _p(x), n_tok, _p(xq), _p(dst), _s())
    return dst


def mmq_compact(ids: torch.Tensor, n_expert: int, x_rows_per_tok: int = 1):
    """-> (bounds [n_expert + 1], ids_src1, ids_dst) of the stable expert sort."""
    n_tok, k = ids.shape
    src = torch.empty(n_tok * k, dtype=torch.int32, device=ids.device)
    dst = torch.empty_like(src)
    bounds = torch.empty(int(lib().fns_hip_mmq_bounds_bytes(n_expert)) // 4, dtype=torch.int32, device=ids.device)
    call("fns_hip_mmq_compact", _p(ids.contiguous()), n_tok, k, n_expert, x_rows_per_tok, _p(src), _p(dst),
         _p(bounds), _s())
    return bounds[: n_expert + 1], src, dst


def mmq_experts(qtype: int, table: torch.Tensor, off: int, ncols: int, nrows: int, n_expert: int, x: torch.Tensor,
                x_rows_per_tok: int, ids: torch.Tensor) -> torch.Tensor:
    """dst [n_tok][n_used][nrows] = W_e . q8_1(x[t][j % x_rows_per_tok])."""
    n_tok, n_used = ids.shape
    x = x.contiguous()
    src = torch.empty(n_tok * n_used, dtype=torch.int32, device=x.device)
    dst_ids = torch.empty_like(src)
    bounds = torch.empty(n_expert + 1, dtype=torch.int32, device=x.device)   # the reference's MmqIdsScratch sizing
    xq = torch.zeros(mmq_q8_1_bytes(ncols, n_tok * x_rows_per_tok), dtype=torch.uint8, device=x.device)
    dst = _empty_f32(n_tok, n_used, nrows, like=x)
    call("fns_hip_mmq_experts", qtype, _p(table), off, ncols, nrows, n_expert, _p(x), x_rows_per_tok, n_tok,
         _p(ids.contiguous()), n_used, _p(src), _p(dst_ids), _p(bounds), _p(xq), _p(dst), _s())
    return dst


def fill_normal(out: torch.Tensor, seed: int, offset: int = 0, mean: float = 0.0, std: float = 1.0) -> torch.Tensor:
    call("fns_hip_fill_normal", _p(out), out.numel(), seed, offset, ctypes.c_float(mean), ctypes.c_float(std), _s())
    return out


def quantize_weights(qtype: int, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """x f32 [..., ncols] on the device -> uint8 [..., row_bytes] GGUF blocks (ggml reference quantisers)."""
    ncols = x.shape[-1]
    nrows = x.numel() // ncols
    if out is None:
        out = torch.empty(*x.shape[:-1], row_bytes(qtype, ncols), dtype=torch.uint8, device=x.device)
    call("fns_hip_quantize_weights", qtype, _p(x.contiguous()), _p(out), nrows, ncols, _s())
    return out


def selftest_lanes() -> int:
    """Bit mask of failing cross-lane exchange checks on the device (0 = all good)."""
    bad = torch.zeros(1, dtype=torch.int32, device="cuda")
    call("fns_hip_selftest_lanes", _p(bad), _s())
    return int(bad.item())


def add(x: torch.Tensor, y: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out = x + y (reference add_inplace, src/kernels.cuh:119); out may be x."""
    out = torch.empty_like(x) if out is None else out
    call("fns_hip_add", _p(x), _p(y), _p(out), x.numel(), _s())
    return out


# The stream of a device as an integer, without the object that torch.cuda.current_stream() makes: a decode step's calls
# are a few microseconds each, and so is what surrounds them here.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _here(what: str, *ts: torch.Tensor | None) -> int:
    """The launch goes to the current device's current stream: every tensor has to be there. -> that stream."""
    dev = torch.cuda.current_device()
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{what}: expected tensors on the current device")
    return _raw_stream(dev)


def add_rms_norm_q8_1(x: torch.Tensor, y: torch.Tensor, w: torch.Tensor, eps: float, sum_out: torch.Tensor | None = None,
                      out: torch.Tensor | None = None, xq: torch.Tensor | None = None):
    """-> (sum, out, xq): sum = x + y, out = RMSNorm(sum) * w, xq its Q8_1 rows. sum_out may be x or y (in place)."""
    shape = x.shape
    n = shape[-1]
    rows = x.numel() // max(n, 1)
    row_bytes_ = (n + 511) // 512 * 576  # q8_1_row_bytes
    if sum_out is None:
        sum_out = torch.empty_like(x)
    if out is None:
        out = torch.empty_like(x)
    if xq is None:
        xq = torch.empty((rows, row_bytes_), dtype=torch.uint8, device=x.device)
    for t in (x, y, sum_out, out):
        if t.dtype != torch.float32 or not t.is_contiguous() or t.shape != shape:
            raise ValueError("add_rms_norm_q8_1: expected contiguous f32 tensors of one shape")
    if w.dtype != torch.float32 or not w.is_contiguous() or w.numel() != n:
        raise ValueError(f"add_rms_norm_q8_1: expected {n} contiguous f32 weights, got {w.numel()} {w.dtype}")
    if xq.dtype != torch.uint8 or not xq.is_contiguous() or xq.numel() != rows * row_bytes_:
        raise ValueError("add_rms_norm_q8_1: xq must be uint8 [rows][q8_1_row_bytes(n)]")
    st = _here("add_rms_norm_q8_1", x, y, w, sum_out, out, xq)
    call("fns_hip_add_rms_norm_q8_1", x.data_ptr(), y.data_ptr(), w.data_ptr(), sum_out.data_ptr(), out.data_ptr(),
         xq.data_ptr(), n, eps, rows, st)
    return sum_out, out, xq


def dequantize_q8_1(xq: torch.Tensor, ncols: int, dtype: torch.dtype = torch.float32):
    """-> (values [nrows][ncols], block sums [nrows][ncols / 32]) that Q8_1 rows stand for, in f32 or f16."""
    if dtype is not torch.float32 and dtype is not torch.float16:
        raise ValueError(f"dequantize_q8_1: {dtype} not supported")
    row_bytes_ = (ncols + 511) // 512 * 576  # q8_1_row_bytes
    if xq.dtype != torch.uint8 or not xq.is_contiguous() or ncols <= 0 or xq.numel() % row_bytes_:
        raise ValueError("dequantize_q8_1: xq must be uint8 [nrows][q8_1_row_bytes(ncols)]")
    st = _here("dequantize_q8_1", xq)
    nrows = xq.numel() // row_bytes_
    x = torch.empty((nrows, ncols), dtype=dtype, device=xq.device)
    sums = torch.empty((nrows, ncols // 32), dtype=dtype, device=xq.device)
    call("fns_hip_dequantize_q8_1", xq.data_ptr(), F32 if dtype is torch.float32 else F16, x.data_ptr(), sums.data_ptr(),
         ncols, nrows, st)
    return x, sums


class KvCacheDesc(ctypes.Structure):
    """Mirror of FnsKvCache (include/fns_hip.h)."""
    _fields_ = [("n_head_kv", ctypes.c_int), ("head_dim", ctypes.c_int), ("page_size", ctypes.c_int),
                ("n_pages", ctypes.c_int64), ("pages", ctypes.c_void_p)]


class KvBatchDesc(ctypes.Structure):
    """Mirror of FnsKvBatch."""
    _fields_ = [("n_seq", ctypes.c_int), ("max_q", ctypes.c_int), ("n_tok", ctypes.c_int64), ("max_kv", ctypes.c_int64),
                ("table_stride", ctypes.c_int64), ("q_start", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("page_table", ctypes.c_void_p)]


class KvAppendDesc(ctypes.Structure):
    """Mirror of FnsKvAppend."""
    _fields_ = [("dtype", ctypes.c_int), ("rope", ctypes.c_int), ("rope_dim", ctypes.c_int), ("n_head", ctypes.c_int),
                ("inv_freq", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("q", ctypes.c_void_p),
                ("q_out", ctypes.c_void_p), ("k_stride", ctypes.c_int64), ("v_stride", ctypes.c_int64),
                ("q_stride", ctypes.c_int64), ("q_out_stride", ctypes.c_int64)]


class AttnDesc(ctypes.Structure):
    """Mirror of FnsAttn."""
    _fields_ = [("dtype", ctypes.c_int), ("n_head", ctypes.c_int), ("window", ctypes.c_int), ("scale", ctypes.c_float),
                ("sinks", ctypes.c_void_p), ("q_stride", ctypes.c_int64), ("out_stride", ctypes.c_int64)]


class KvTreeDesc(ctypes.Structure):
    """Mirror of FnsKvTree."""
    _fields_ = [("sees", ctypes.c_void_p), ("words", ctypes.c_int)]


class KvEvictDesc(ctypes.Structure):
    """Mirror of FnsKvEvict."""
    _fields_ = [("budget", ctypes.c_int), ("first", ctypes.c_int), ("recent", ctypes.c_int), ("weights", ctypes.c_void_p),
                ("weights_out", ctypes.c_void_p), ("to_table", ctypes.c_void_p), ("to_stride", ctypes.c_int64),
                ("kept", ctypes.c_void_p), ("new_len", ctypes.c_void_p), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_size_t)]


class KvKeepDesc(ctypes.Structure):
    """Mirror of FnsKvKeep."""
    _fields_ = [("kept", ctypes.c_void_p), ("n_kept", ctypes.c_void_p), ("stride", ctypes.c_int64),
                ("weights", ctypes.c_void_p), ("new_len", ctypes.c_void_p)]


class KvCache:
    """A paged key/value cache held in 4 bits (FnsKvCache): n_pages pages of page_size positions of every kv head, one
    layer's. pages: uint8 device memory of an earlier cache of this shape, or None: zeroed."""

    def __init__(self, n_pages: int, page_size: int, n_head_kv: int, head_dim: int, pages: torch.Tensor | None = None):
        self.page_bytes = int(lib().fns_hip_kv_page_bytes(n_head_kv, head_dim, page_size))
        if not self.page_bytes or n_pages <= 0:
            raise ValueError(f"KvCache: unsupported shape (n_pages {n_pages}, page_size {page_size}, n_head_kv {n_head_kv}, "
                             f"head_dim {head_dim})")
        if pages is None:
            pages = torch.zeros(n_pages, self.page_bytes, dtype=torch.uint8, device="cuda")
        if pages.dtype != torch.uint8 or not pages.is_contiguous() or pages.numel() != n_pages * self.page_bytes:
            raise ValueError(f"KvCache: pages must be contiguous uint8 of {n_pages} * {self.page_bytes} bytes")
        _here("KvCache", pages)
        self.pages, self.n_head_kv, self.head_dim, self.page_size = pages, n_head_kv, head_dim, page_size
        self.desc = KvCacheDesc(n_head_kv, head_dim, page_size, n_pages, pages.data_ptr())
        self.ref = ctypes.byref(self.desc)


class KvBatch:
    """New tokens of some sequences over a KvCache (FnsKvBatch): q_start [n_seq + 1], kv_len [n_seq] and page_table
    [n_seq][pages of a sequence] int32 device tensors, whose values a captured graph takes anew at each replay; n_tok rows of
    the token arrays, max_q at least the new tokens of any sequence, max_kv about the longest sequence, by which attn divides its
    work (None: what the table has room for; results are right, but far shorter contexts than that are divided badly)."""

    def __init__(self, q_start: torch.Tensor, kv_len: torch.Tensor, page_table: torch.Tensor, n_tok: int, max_q: int,
                 max_kv: int | None = None):
        n_seq = kv_len.numel()
        for t in (q_start, kv_len, page_table):
            if t.dtype != torch.int32 or not t.is_contiguous():
                raise ValueError("KvBatch: expected contiguous int32 tensors")
        if q_start.numel() != n_seq + 1 or page_table.dim() != 2 or page_table.shape[0] != n_seq:
            raise ValueError("KvBatch: expected q_start [n_seq + 1], kv_len [n_seq] and page_table [n_seq][pages]")
        _here("KvBatch", q_start, kv_len, page_table)
        self.q_start, self.kv_len, self.page_table, self.n_tok = q_start, kv_len, page_table, n_tok
        self._open = max_kv is None  # the table's room, which depends on the cache's page size
        self.desc = KvBatchDesc(n_seq, max_q, n_tok, max_kv or 0, page_table.shape[1], q_start.data_ptr(), kv_len.data_ptr(),
                                page_table.data_ptr())
        self.ref = ctypes.byref(self.desc)

    def _for(self, cache: KvCache):
        if self._open:
            self.desc.max_kv = min(self.desc.table_stride * cache.page_size, 2 ** 31 - 1)
        return self.ref

    @classmethod
    def from_lists(cls, q_lens, kv_lens, pages, n_tok: int | None = None) -> "KvBatch":
        """From host lists: new tokens and lengths (with them) of every sequence, and its pages in order."""
        start = [0]
        for q in q_lens:
            start.append(start[-1] + q)
        width = max([len(p) for p in pages] + [1])
        table = [list(p) + [-1] * (width - len(p)) for p in pages]
        dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        return cls(dev(start), dev(list(kv_lens)), dev(table).view(len(table), width), start[-1] if n_tok is None else n_tok,
                   max([*q_lens, 0]), max([*kv_lens, 0]))


def rope_freqs(rope_dim: int, base: float = 10000.0, factors=None) -> torch.Tensor:
    """inv_freq of kv_append: base^(-2 i / rope_dim), divided by factors[i] if given; f32 on the current device."""
    f = float(base) ** (-torch.arange(0, rope_dim, 2, dtype=torch.float64) / rope_dim)
    if factors is not None:
        f = f / torch.as_tensor(factors, dtype=torch.float64, device="cpu")
    return f.float().cuda()


def rope_scaled(rope_dim: int, base: float, factor: float, original: float, fast: float = 32.0, slow: float = 1.0):
    """-> (inv_freq f32 on the current device, magnitude) of kv_append for contexts of factor * original positions: pairs that
    turn `fast` times or more over the original ones keep their frequency, those that turn `slow` times or less have it divided
    by factor (fns_hip_rope_scaled)."""
    if rope_dim <= 0 or rope_dim % 2:
        raise ValueError(f"rope_scaled: an even rope_dim is needed ({rope_dim})")
    freq, magnitude = (ctypes.c_float * (rope_dim // 2))(), ctypes.c_float()
    call("fns_hip_rope_scaled", rope_dim, base, factor, original, fast, slow, freq, ctypes.byref(magnitude))
    return torch.tensor(list(freq), dtype=torch.float32).cuda(), magnitude.value


class KvTree:
    """What the new tokens of a batch see of their sequence's new tokens (FnsKvTree): sees int64 [n_tok][words], bit j % 64 of
    word j / 64 for the j-th of them; pos int32 [n_tok] or None, the positions that kv_append may turn them by."""

    def __init__(self, sees: torch.Tensor, pos: torch.Tensor | None = None):
        if sees.dtype != torch.int64 or not sees.is_contiguous() or sees.dim() != 2:
            raise ValueError("KvTree: sees must be contiguous int64 [n_tok][words]")
        _here("KvTree", sees, pos)
        self._set(sees, pos)

    def _set(self, sees: torch.Tensor, pos: torch.Tensor | None) -> "KvTree":
        self.sees, self.pos = sees, pos
        self.desc = KvTreeDesc(sees.data_ptr(), sees.shape[1])
        self.ref = ctypes.byref(self.desc)
        return self

    def _for(self, what: str, batch: KvBatch):
        if self.sees.shape[0] != batch.n_tok:
            raise ValueError(f"{what}: the tree has {self.sees.shape[0]} tokens, the batch {batch.n_tok}")
        return self.ref


def _ints(what: str, name: str, t: torch.Tensor, *shape: int) -> int:
    if t.dtype != torch.int32 or not t.is_contiguous() or tuple(t.shape) != shape:
        raise ValueError(f"{what}: {name} must be contiguous int32 {list(shape)}")
    return t.data_ptr()


def tree_plan(batch: KvBatch, parents: torch.Tensor, base: torch.Tensor | None = None, words: int | None = None) -> KvTree:
    """The tree of the batch's new tokens from parents int32 [n_tok] (index among the sequence's new tokens, -1: none, anything
    below: no token of the tree), with positions base[sequence] (None: the sequence's first new position) + number of
    ancestors. words: 64-bit words a token (None: as max_q needs)."""
    if words is None:
        words = max(1, (batch.desc.max_q + 63) // 64)
    p = _ints("tree_plan", "parents", parents, batch.n_tok)
    b = None if base is None else _ints("tree_plan", "base", base, batch.desc.n_seq)
    sees = parents.new_empty((batch.n_tok, max(words, 0)), dtype=torch.int64)
    pos = parents.new_empty(batch.n_tok)
    st = _here("tree_plan", batch.kv_len, parents, base)
    call("fns_hip_tree_plan", batch.ref, p, b, words, sees.data_ptr(), pos.data_ptr(), st)
    return KvTree.__new__(KvTree)._set(sees, pos)


def _heads(what: str, t: torch.Tensor, n_tok: int, dim: int, dtype: torch.dtype) -> int:
    """Token stride of t [n_tok][heads][dim], heads contiguous within a token (a slice of a fused projection is)."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != n_tok or shape[2] != dim:
        raise ValueError(f"{what}: expected [{n_tok}][heads][{dim}], got {list(shape)}")
    if t.dtype is not dtype or (dtype is not torch.float32 and dtype is not torch.bfloat16):
        raise ValueError(f"{what}: expected one type of f32 and bf16, got {t.dtype}")
    width = shape[1] * dim
    if t.is_contiguous():
        return width
    s0, s1, s2 = t.stride()
    if s2 != 1 or (shape[1] > 1 and s1 != dim):
        raise ValueError(f"{what}: the heads of a token must be contiguous")
    if n_tok <= 1:
        return width
    if s0 < width:
        raise ValueError(f"{what}: tokens overlap")
    return s0


def kv_append(cache: KvCache, batch: KvBatch, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None,
              rope: int = ROPE_NONE, inv_freq: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
              pos: torch.Tensor | None = None, magnitude: float = 1.0):
    """k, v [n_tok][n_head_kv][head_dim] into the cache, k (and q) rotated by position * inv_freq over the first
    2 * len(inv_freq) channels. pos int32 [n_tok]: positions to turn by (None: those in the cache); magnitude: of what is
    rotated. -> the rotated q (in q_out, which may be q; None without q)."""
    D, Hk, n_tok, dt = cache.head_dim, cache.n_head_kv, batch.n_tok, k.dtype
    x = KvAppendDesc()
    x.k_stride, x.v_stride = _heads("kv_append", k, n_tok, D, dt), _heads("kv_append", v, n_tok, D, dt)
    if k.shape[1] != Hk or v.shape[1] != Hk:
        raise ValueError(f"kv_append: expected {Hk} kv heads, got {k.shape[1]} and {v.shape[1]}")
    if q is not None:
        if q_out is None:
            q_out = q.new_empty(q.shape, dtype=dt)
        x.q_stride = _heads("kv_append", q, n_tok, D, dt)
        x.q_out_stride = _heads("kv_append", q_out, n_tok, D, dt)
        if q_out.shape != q.shape:
            raise ValueError("kv_append: q_out is not of q's shape")
        x.n_head, x.q, x.q_out = q.shape[1], q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("kv_append: q_out without q")
    if rope != ROPE_NONE:
        if inv_freq is None or inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous() or inv_freq.dim() != 1:
            raise ValueError("kv_append: a rotation needs inv_freq, a contiguous f32 vector")
        x.rope, x.rope_dim, x.inv_freq = rope, 2 * inv_freq.numel(), inv_freq.data_ptr()
    else:
        inv_freq = None
    x.dtype, x.k, x.v = F32 if dt is torch.float32 else BF16, k.data_ptr(), v.data_ptr()
    st = _here("kv_append", cache.pages, batch.kv_len, k, v, q, q_out, inv_freq, pos)
    if pos is None and magnitude == 1.0:
        call("fns_hip_kv_append", cache.ref, batch._for(cache), ctypes.byref(x), st)
    else:
        at = None if pos is None else _ints("kv_append", "pos", pos, n_tok)
        call("fns_hip_kv_append_at", cache.ref, batch._for(cache), ctypes.byref(x), at, magnitude, st)
    return q_out


def kv_read(cache: KvCache, batch: KvBatch):
    """-> (k, v) f32 [n_tok][n_head_kv][head_dim]: what the cache holds of the batch's tokens."""
    st = _here("kv_read", cache.pages, batch.kv_len)
    shape = (batch.n_tok, cache.n_head_kv, cache.head_dim)
    k = cache.pages.new_empty(shape, dtype=torch.float32)
    v = k.new_empty(shape)
    call("fns_hip_kv_read", cache.ref, batch._for(cache), k.data_ptr(), v.data_ptr(), st)
    return k, v


def attn_workspace(cache: KvCache, batch: KvBatch, q: torch.Tensor) -> torch.Tensor:
    """A workspace of attn (with or without a tree) for this batch's numbers and q's heads; it may serve every layer of a step
    in turn."""
    width = _heads("attn", q, batch.n_tok, cache.head_dim, q.dtype)
    desc = AttnDesc(_dtype_code(q), q.shape[1], 0, 1.0, None, width, q.shape[1] * cache.head_dim)
    size = ctypes.c_size_t()
    call("fns_hip_attn_tree_workspace", cache.ref, batch._for(cache), ctypes.byref(desc), ctypes.byref(size))
    return torch.empty(size.value, dtype=torch.uint8, device=q.device)


def attn(cache: KvCache, batch: KvBatch, q: torch.Tensor, scale: float | None = None, window: int = 0,
         sinks: torch.Tensor | None = None, out: torch.Tensor | None = None, ws: torch.Tensor | None = None,
         tree: KvTree | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of q [n_tok][n_head][head_dim] over the cache -> out (rows of no sequence are left as they were). scale
    None: head_dim^-0.5; window > 0: the last `window` positions only; sinks f32 [n_head] join the denominator. tree: what the
    new tokens see of each other; lse f32 [n_tok][n_head]: takes the logarithms of the denominators (kv_weigh's; of a row
    that sees nothing the sink, or -infinity)."""
    D, dt = cache.head_dim, q.dtype
    if out is None:
        out = torch.empty(q.shape, dtype=dt, device=q.device)
    desc = AttnDesc()
    desc.q_stride, desc.out_stride = _heads("attn", q, batch.n_tok, D, dt), _heads("attn", out, batch.n_tok, D, dt)
    if out.shape != q.shape:
        raise ValueError("attn: out is not of q's shape")
    if sinks is not None:
        if sinks.dtype != torch.float32 or not sinks.is_contiguous() or sinks.numel() != q.shape[1]:
            raise ValueError("attn: sinks must be a contiguous f32 vector, one a query head")
        desc.sinks = sinks.data_ptr()
    desc.dtype, desc.n_head, desc.window = F32 if dt is torch.float32 else BF16, q.shape[1], min(window, 2 ** 31 - 1)
    desc.scale = D ** -0.5 if scale is None else scale
    if ws is None:
        ws = attn_workspace(cache, batch, q)
    elif not ws.is_contiguous():
        raise ValueError("attn: the workspace must be contiguous")
    st = _here("attn", cache.pages, batch.kv_len, q, out, sinks, ws, lse, None if tree is None else tree.sees)
    if tree is not None or lse is not None:
        if lse is not None and (lse.dtype != torch.float32 or not lse.is_contiguous() or lse.shape != q.shape[:2]):
            raise ValueError("attn: lse must be contiguous f32 [n_tok][n_head]")
        call("fns_hip_attn_tree", cache.ref, batch._for(cache), ctypes.byref(desc), None if tree is None else tree._for("attn", batch),
             q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel() * ws.element_size(), st)
        return out
    call("fns_hip_attn", cache.ref, batch._for(cache), ctypes.byref(desc), q.data_ptr(), out.data_ptr(), ws.data_ptr(),
         ws.numel() * ws.element_size(), st)
    return out


def kv_weights(cache: KvCache) -> torch.Tensor:
    """Zeroed attention weights of a cache's positions: f32 [n_pages][n_head_kv][page_size]."""
    return torch.zeros(cache.desc.n_pages, cache.n_head_kv, cache.page_size, dtype=torch.float32, device=cache.pages.device)


def _weights(what: str, cache: KvCache, *ts: torch.Tensor | None) -> None:
    shape = (cache.desc.n_pages, cache.n_head_kv, cache.page_size)
    for t in ts:
        if t is not None and (t.dtype != torch.float32 or not t.is_contiguous() or tuple(t.shape) != shape):
            raise ValueError(f"{what}: weights must be contiguous f32 {list(shape)}")


def kv_weigh_workspace(cache: KvCache, batch: KvBatch, q: torch.Tensor) -> torch.Tensor:
    """A workspace of kv_weigh for this batch's numbers and q's heads; it may serve every layer of a step in turn."""
    width = _heads("kv_weigh", q, batch.n_tok, cache.head_dim, q.dtype)
    desc = AttnDesc(_dtype_code(q), q.shape[1], 0, 1.0, None, width, 0)
    size = ctypes.c_size_t()
    call("fns_hip_kv_weigh_workspace", cache.ref, batch._for(cache), ctypes.byref(desc), ctypes.byref(size))
    return torch.empty(size.value, dtype=torch.uint8, device=q.device)


def kv_weigh(cache: KvCache, batch: KvBatch, q: torch.Tensor, lse: torch.Tensor, past: torch.Tensor | None,
             scale: float | None = None, window: int = 0, tree: KvTree | None = None, out: torch.Tensor | None = None,
             ws: torch.Tensor | None = None) -> torch.Tensor:
    """What every cached position (of sequences with new tokens) gets of the new tokens' attention, exp(scale * q . K - lse)
    summed over tokens and the heads of a group, on top of `past` (as kv_weights; None: zeros; new positions start at 0) -> out
    (None: past, in place). lse as attn gives it; rows whose lse is not finite add nothing."""
    if out is None:
        out = kv_weights(cache) if past is None else past
    _weights("kv_weigh", cache, past, out)
    D, dt = cache.head_dim, q.dtype
    desc = AttnDesc(F32 if dt is torch.float32 else BF16, q.shape[1], min(window, 2 ** 31 - 1), D ** -0.5 if scale is None else scale,
                    None, _heads("kv_weigh", q, batch.n_tok, D, dt), 0)
    if lse.dtype != torch.float32 or not lse.is_contiguous() or lse.shape != q.shape[:2]:
        raise ValueError("kv_weigh: lse must be contiguous f32 [n_tok][n_head]")
    if ws is None:
        ws = kv_weigh_workspace(cache, batch, q)
    elif not ws.is_contiguous():
        raise ValueError("kv_weigh: the workspace must be contiguous")
    st = _here("kv_weigh", cache.pages, batch.kv_len, q, lse, past, out, ws, None if tree is None else tree.sees)
    call("fns_hip_kv_weigh", cache.ref, batch._for(cache), ctypes.byref(desc), None if tree is None else tree._for("kv_weigh", batch),
         q.data_ptr(), lse.data_ptr(), None if past is None else past.data_ptr(), out.data_ptr(), ws.data_ptr(),
         ws.numel() * ws.element_size(), st)
    return out


def kv_evict_workspace(cache: KvCache, batch: KvBatch) -> torch.Tensor | None:
    """A workspace of kv_evict for this batch's numbers; None where it needs none (tables of up to 32768 positions)."""
    if batch.desc.table_stride * cache.page_size <= 32768:
        return None
    size = ctypes.c_size_t()
    call("fns_hip_kv_evict_workspace", cache.ref, batch._for(cache), ctypes.byref(size))
    return torch.empty(size.value, dtype=torch.uint8, device=cache.pages.device)


def kv_evict(cache: KvCache, batch: KvBatch, weights: torch.Tensor, budget: int, first: int = 0, recent: int = 0,
             to_table: torch.Tensor | None = None, weights_out: torch.Tensor | None = None, ws: torch.Tensor | None = None):
    """Cuts every sequence to `budget` positions a kv head: the first `first`, the last `recent`, and of the others those of the
    largest weights; K, V and weights of the kept ones move to the front of the sequence, in order: of its own pages, or of
    to_table's int32 [n_seq][pages] (weights_out: None: weights). -> (kept int32 [n_seq][n_head_kv][budget], the kept positions and
    then -1; new_len int32 [n_seq])."""
    if weights_out is None:
        weights_out = weights
    _weights("kv_evict", cache, weights, weights_out)
    if max(abs(budget), abs(first), abs(recent)) > 1 << 30:  # (they would wrap in the descriptor)
        raise ValueError(f"kv_evict: budget must be 1..2^30 and hold first and recent ({budget}, {first}, {recent})")
    n_seq = batch.desc.n_seq
    kept = batch.kv_len.new_empty((n_seq, cache.n_head_kv, max(budget, 0)))
    new_len = batch.kv_len.new_empty(n_seq)
    x = KvEvictDesc(budget, first, recent, weights.data_ptr(), weights_out.data_ptr(), None, 0, kept.data_ptr(), new_len.data_ptr())
    if to_table is not None:
        if to_table.dim() != 2:
            raise ValueError("kv_evict: to_table must be [n_seq][pages]")
        x.to_table, x.to_stride = _ints("kv_evict", "to_table", to_table, n_seq, to_table.shape[1]), to_table.shape[1]
    if ws is None:
        ws = kv_evict_workspace(cache, batch)
    elif not ws.is_contiguous():
        raise ValueError("kv_evict: the workspace must be contiguous")
    if ws is not None:
        x.workspace, x.workspace_bytes = ws.data_ptr(), ws.numel() * ws.element_size()
    st = _here("kv_evict", cache.pages, batch.kv_len, weights, weights_out, to_table, ws)
    call("fns_hip_kv_evict", cache.ref, batch._for(cache), ctypes.byref(x), st)
    return kept, new_len


def kv_keep(cache: KvCache, batch: KvBatch, kept: torch.Tensor, n_kept: torch.Tensor, weights: torch.Tensor | None = None) -> torch.Tensor:
    """Of every sequence's new tokens the listed ones (kept int32 [n_seq][most], the first n_kept[s] of a row, indices among the
    sequence's new tokens) become its next positions, in the list's order; weights (as kv_weights) move along.
    -> new_len int32 [n_seq]."""
    _weights("kv_keep", cache, weights)
    n_seq = batch.desc.n_seq
    if kept.dim() != 2:
        raise ValueError("kv_keep: kept must be [n_seq][most]")
    new_len = n_kept.new_empty(n_seq, dtype=torch.int32)
    x = KvKeepDesc(_ints("kv_keep", "kept", kept, n_seq, kept.shape[1]), _ints("kv_keep", "n_kept", n_kept, n_seq), kept.shape[1],
                   None if weights is None else weights.data_ptr(), new_len.data_ptr())
    st = _here("kv_keep", cache.pages, batch.kv_len, kept, n_kept, weights)
    call("fns_hip_kv_keep", cache.ref, batch._for(cache), ctypes.byref(x), st)
    return new_len


class DenseFfnDesc(ctypes.Structure):
    _fields_ = [("hidden", ctypes.c_int), ("inter", ctypes.c_int), ("gate_type", ctypes.c_int),
                ("up_type", ctypes.c_int), ("down_type", ctypes.c_int), ("gate", ctypes.c_void_p),
                ("up", ctypes.c_void_p), ("down", ctypes.c_void_p), ("ffn_norm", ctypes.c_void_p),
                ("norm_eps", ctypes.c_float)]


class DenseFfn:
    """A dense FFN layer (the reference model's leading dense blocks, src/engine.cu:655-667 decode and :331-337
    prefill): out = x + down . q8_1(silu(gate . q8_1(h)) * (up . q8_1(h))), h = RMSNorm(x) * ffn_norm."""

    def __init__(self, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, gate_type: int, up_type: int,
                 down_type: int, hidden: int, inter: int, ffn_norm: torch.Tensor | None = None,
                 norm_eps: float = 1e-6):
        self.gate, self.up, self.down, self.ffn_norm = gate, up, down, ffn_norm
        self.desc = DenseFfnDesc(hidden, inter, gate_type, up_type, down_type, gate.data_ptr(), up.data_ptr(),
                                 down.data_ptr(), ffn_norm.data_ptr() if ffn_norm is not None else None, norm_eps)

    @classmethod
    def from_gguf(cls, file: "GgufFile", layer: int) -> "DenseFfn":
        """Dense layer `layer` of a GGUF checkpoint made resident by fns_hip_dense_ffn_from_gguf."""
        obj = cls.__new__(cls)
        obj.desc = DenseFfnDesc()
        obj.gate = obj.up = obj.down = obj.ffn_norm = None
        obj._file = file
        res = ctypes.c_void_p()
        call("fns_hip_dense_ffn_from_gguf", file.handle, layer, ctypes.byref(res), ctypes.byref(obj.desc))
        obj._resident = res
        return obj

    def __del__(self):
        res = getattr(self, "_resident", None)
        if res:
            lib().fns_hip_dense_resident_free(res)
            self._resident = None

    def workspace(self, n_tok: int) -> torch.Tensor:
        total = ctypes.c_size_t()
        call("fns_hip_dense_ffn_workspace", ctypes.byref(self.desc), n_tok, ctypes.byref(total))
        return torch.empty(total.value, dtype=torch.uint8, device="cuda")

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None, ws: torch.Tensor | None = None,
                 prefill: bool = False) -> torch.Tensor:
        x = x.contiguous()
        n_tok = x.numel() // self.desc.hidden
        out = torch.empty_like(x) if out is None else out
        ws = self.workspace(n_tok) if ws is None else ws
        call("fns_hip_dense_ffn_prefill" if prefill else "fns_hip_dense_ffn", ctypes.byref(self.desc), _p(x),
             _p(out), n_tok, _p(ws), ws.numel(), _s())
        return out


class GgufTensorInfo(ctypes.Structure):
    """Mirror of FnsGgufTensorInfo (include/fns_hip.h)."""
    _fields_ = [("type", ctypes.c_int), ("n_dims", ctypes.c_int), ("ne", ctypes.c_int64 * 4),
                ("nbytes", ctypes.c_size_t), ("offset", ctypes.c_size_t), ("data", ctypes.c_void_p)]


class GgufFile:
    """A GGUF checkpoint mapped by the library's reader (fns_hip_gguf_*; reference src/model.cpp:30-136)."""

    def __init__(self, path: str):
        self.handle = None
        h = ctypes.c_void_p()
        call("fns_hip_gguf_open", str(path).encode(), ctypes.byref(h))
        self.handle = h

    def close(self) -> None:
        if getattr(self, "handle", None):
            lib().fns_hip_gguf_close(self.handle)
            self.handle = None

    def __del__(self):
        self.close()

    def info(self) -> dict:
        v, nt, nk, off = ctypes.c_uint32(), ctypes.c_int64(), ctypes.c_int64(), ctypes.c_size_t()
        call("fns_hip_gguf_info", self.handle, ctypes.byref(v), ctypes.byref(nt), ctypes.byref(nk), ctypes.byref(off))
        return {"version": v.value, "n_tensors": nt.value, "n_kv": nk.value, "data_offset": off.value}

    def tensor(self, name: str) -> dict:
        info = GgufTensorInfo()
        call("fns_hip_gguf_tensor", self.handle, name.encode(), ctypes.byref(info))
        return self._as_dict(info)

    def tensors(self) -> list[tuple[str, dict]]:
        out = []
        for i in range(self.info()["n_tensors"]):
            info, name = GgufTensorInfo(), ctypes.c_char_p()
            call("fns_hip_gguf_tensor_at", self.handle, i, ctypes.byref(info), ctypes.byref(name))
            out.append((name.value.decode(), self._as_dict(info)))
        return out

    @staticmethod
    def _as_dict(info: GgufTensorInfo) -> dict:
        raw = (ctypes.c_uint8 * info.nbytes).from_address(info.data) if info.nbytes else b""
        return {"type": info.type, "ne": list(info.ne[: info.n_dims]), "nbytes": info.nbytes, "offset": info.offset,
                "bytes": np.frombuffer(raw, dtype=np.uint8).copy() if info.nbytes else np.zeros(0, np.uint8)}

    def u32(self, key: str) -> int:
        v = ctypes.c_uint32()
        call("fns_hip_gguf_get_u32", self.handle, key.encode(), ctypes.byref(v))
        return v.value

    def f32(self, key: str) -> float:
        v = ctypes.c_float()
        call("fns_hip_gguf_get_f32", self.handle, key.encode(), ctypes.byref(v))
        return v.value

    def bool(self, key: str) -> bool:
        v = ctypes.c_int()
        call("fns_hip_gguf_get_bool", self.handle, key.encode(), ctypes.byref(v))
        return bool(v.value)

    def str(self, key: str) -> str:
        v = ctypes.c_char_p()
        call("fns_hip_gguf_get_str", self.handle, key.encode(), ctypes.byref(v))
        return v.value.decode()
