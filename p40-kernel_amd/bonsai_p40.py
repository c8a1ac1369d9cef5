"""Host-side Python binding of libbonsai_p40.so (the gfx950 PQ2_0 matmul path).

The native library exports the C ABI of include/bonsai_p40.h; this module
binds it with ctypes and offers thin wrappers over torch device tensors
(torch is used only for device memory and the current HIP stream).  Every
wrapper raises if the library is missing or a call returns nonzero -- there is
no CPU fallback in this module.

Reference interface mirrored: include/bonsai_p40.h of boetti-dev/p40-kernel
(bonsai_p40_gemv, _quant_activations, _gemm, _repack, _gemv_repack, _fwht,
_rmsnorm), plus the additions declared at the end of the header.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libbonsai_p40.so")

QK_PQ2 = 128          # weights per block_pq2_0
QK8 = 32              # elements per block_q8_1
PQ2_BYTES = 34        # sizeof(block_pq2_0)
Q81_BYTES = 36        # sizeof(block_q8_1)
HBLK = 1024           # Hadamard block

# Every symbol of include/bonsai_p40.h with its ctypes signature.
_V, _I64, _F32P = C.c_void_p, C.c_int64, C.c_void_p
SIGNATURES = {
    "bonsai_p40_gemv": [_V, _V, _F32P, _I64, _I64, _V],
    "bonsai_p40_quant_activations": [_F32P, _V, _I64, _V],
    "bonsai_p40_gemm": [_V, _V, _F32P, _I64, _I64, _I64, _V],
    "bonsai_p40_gemm_ws": [_V, _V, _F32P, _I64, _I64, _I64, _V, _I64, _V],
    "bonsai_p40_gemm_workspace_bytes": [_I64, _I64],
    "bonsai_p40_repack": [_V, _V, _I64, _I64, _V],
    "bonsai_p40_gemv_repack": [_V, _F32P, _F32P, _I64, _I64, _V],
    "bonsai_p40_fwht": [_F32P, _F32P, _I64, _V],
    "bonsai_p40_fwht_signs_n": [_F32P, _F32P, _I64, _V],
    "bonsai_p40_rmsnorm": [_F32P, _F32P, _F32P, _I64, _I64, C.c_float, _V],
    "bonsai_p40_gdn_step": [_F32P] * 7 + [C.c_int] * 4 + [_V],
    "bonsai_p40_attn": [_F32P] * 4 + [C.c_int] * 4 + [C.c_float, _V],
    "bonsai_p40_fwht_quant": [_F32P, _F32P, _V, _I64, _V],
    "bonsai_p40_quant_tokens": [_F32P, _F32P, _V, _I64, _I64, C.c_int, _V],
    "bonsai_p40_swiglu_fwht_quant": [_F32P, _F32P, _F32P, _V, _I64, _V],
    "bonsai_p40_rmsnorm_fwht_quant": [_F32P, _F32P, _F32P, _V, _I64, _I64, C.c_float, _V],
    "bonsai_p40_fwht_gemv": [_V, _F32P, _F32P, _F32P, _I64, _I64, _V],
    "bonsai_p40_quant_gemv": [_V, _F32P, _F32P, _I64, _I64, _V],
    "bonsai_p40_ggml_should_use": [C.c_int, C.c_int, _I64],
    "bonsai_p40_ggml_mul_mat": [_V, _V, _V, _V, C.c_size_t, _V],
    "bonsai_p40_gemv_group": [_V, _V, _V, C.c_int, _V, _I64, _V],
    "bonsai_p40_fwht_gemv_group": [_V, _V, _V, C.c_int, _F32P, _F32P, _I64, _V],
    "bonsai_p40_rmsnorm_fwht_gemv_group": [_V, _V, _V, C.c_int, _F32P, _F32P, _F32P, _I64, C.c_float, _V],
    "bonsai_p40_ffn_gate_up_swiglu": [_V, _V, _F32P, _F32P, _F32P, _F32P, _V, _I64, _I64, C.c_float, _V, _V, _V],
    "bonsai_p40_ffn_gate_up_swiglu_noalloc": [_V, _V, _F32P, _F32P, _F32P, _F32P, _V, _I64, _I64, C.c_float,
                                              _V, _V],
    "bonsai_p40_quantize_pq2_0": [_F32P, _V, _I64, _V],
    "bonsai_p40_dequantize_pq2_0": [_V, _F32P, _I64, _V],
    "bonsai_p40_qk_norm_rope": [_V, _V],
    "bonsai_p40_attn_paged": [_V, _V],
    "bonsai_p40_attn_paged_workspace_bytes": [_V],
    "bonsai_p40_attn_shared": [_V, _V],
    "bonsai_p40_attn_shared_workspace_bytes": [_V],
    "bonsai_p40_kv_read": [_V, _V],
    "bonsai_p40_gdn": [_V, _V],
    "bonsai_p40_gdn_workspace_bytes": [_V],
    "bonsai_p40_chunk_dots": [_V, _V, _V, _I64, _I64, _V],
    "bonsai_p40_stream_read": [_V, _I64, _V, C.c_int, _V],
    "bonsai_p40_reload_tuning": [],
    "bonsai_p40_mfma_probe": [C.c_int, C.c_int, C.c_int, _V, _V, _V],
    "bonsai_p40_overlap_probe": [C.c_int, C.c_int, C.c_int, C.c_int, _V, _V],
    "bonsai_p40_launch_probe": [C.c_int, C.c_int, _V, _V],
    "bonsai_p40_unit_dma_probe": [_V, _I64, _I64, _V, _V],
    "bonsai_p40_chain_plan_bytes": [C.c_int],
    "bonsai_p40_chain_plan": [_V, C.c_int, _V],
    "bonsai_p40_chain_run": [_V, C.c_int, _V, _V, _V],
}
RESTYPES = {"bonsai_p40_chain_plan_bytes": C.c_int64, "bonsai_p40_gemm_workspace_bytes": C.c_int64,
            "bonsai_p40_attn_paged_workspace_bytes": C.c_int64, "bonsai_p40_attn_shared_workspace_bytes": C.c_int64,
            "bonsai_p40_gdn_workspace_bytes": C.c_int64}

_lib = None


def lib() -> C.CDLL:
    """Load libbonsai_p40.so; raise if it was not built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `make -C p40-kernel_amd` "
                "(or __graft_entry__.build())")
        L = C.CDLL(LIB_PATH)
        for name, argtypes in SIGNATURES.items():
            fn = getattr(L, name)
            fn.argtypes = argtypes
            fn.restype = RESTYPES.get(name, C.c_int)
        _lib = L
    return _lib


class BonsaiError(RuntimeError):
    pass


def _check(name: str, rc: int) -> None:
    if rc != 0:
        raise BonsaiError(f"{name} returned {rc}")


def _ptr(t) -> int | None:
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


_raw_stream = _device = None     # a device's current stream as a hipStream_t; the current device


def _init_streams() -> None:
    global _raw_stream, _device
    import torch
    torch.cuda.current_stream()                           # initialises the device
    # what torch.cuda.current_stream(dev).cuda_stream comes to, without the objects made on the way (0.2 us, not 2.9)
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
        lambda dev: torch.cuda.current_stream(dev).cuda_stream)
    _device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _stream(stream) -> int | None:
    if stream is not None:
        return stream if isinstance(stream, int) else stream.cuda_stream
    if _device is None:
        _init_streams()
    return _raw_stream(_device())


def call(name: str, *args, stream=None) -> int:
    """Raw call: tensors are passed as device pointers; returns the rc."""
    fn = getattr(lib(), name)
    conv = [_ptr(a) if (a is None or hasattr(a, "data_ptr")) else a for a in args]
    return fn(*conv, _stream(stream))


# -------------------------------------------------------------- wrappers
def gemv(W, xq, y, n_out: int, n_in: int, stream=None) -> None:
    _check("bonsai_p40_gemv", call("bonsai_p40_gemv", W, xq, y, n_out, n_in, stream=stream))


def quant_activations(x, out, n: int, stream=None) -> None:
    _check("bonsai_p40_quant_activations",
           call("bonsai_p40_quant_activations", x, out, n, stream=stream))


def gemm(W, Xq, Y, n_out: int, n_in: int, n_tok: int, stream=None) -> None:
    _check("bonsai_p40_gemm", call("bonsai_p40_gemm", W, Xq, Y, n_out, n_in, n_tok, stream=stream))


def gemm_workspace_bytes(n_in: int, n_tok: int) -> int:
    """bonsai_p40_gemm_workspace_bytes: the workspace bonsai_p40_gemm_ws needs."""
    return int(lib().bonsai_p40_gemm_workspace_bytes(n_in, n_tok))


def gemm_ws(W, Xq, Y, n_out: int, n_in: int, n_tok: int, ws, ws_bytes=None, stream=None) -> None:
    """bonsai_p40_gemm with a workspace (a tensor, or a pointer with ws_bytes);
    Y is bit-identical to gemm()'s."""
    if ws_bytes is None:
        ws_bytes = 0 if ws is None else ws.numel() * ws.element_size()
    _check("bonsai_p40_gemm_ws", call("bonsai_p40_gemm_ws", W, Xq, Y, n_out, n_in, n_tok, ws, ws_bytes,
                                      stream=stream))


def repack(src, dst, n_out: int, n_in: int, stream=None) -> None:
    _check("bonsai_p40_repack", call("bonsai_p40_repack", src, dst, n_out, n_in, stream=stream))


def gemv_repack(W, x, y, n_out: int, n_in: int, stream=None) -> None:
    _check("bonsai_p40_gemv_repack",
           call("bonsai_p40_gemv_repack", W, x, y, n_out, n_in, stream=stream))


def fwht(x, signs, n: int, stream=None) -> None:
    """In-place FWHT-1024 blocks; signs (or None) has 1024 entries reused by
    every block, as the reference device kernel."""
    _check("bonsai_p40_fwht", call("bonsai_p40_fwht", x, signs, n, stream=stream))


def fwht_signs_n(x, signs, n: int, stream=None) -> None:
    """In-place FWHT-1024 blocks; signs (or None) is a length-n vector, block
    b using signs[1024 b ..] (the host fwht_blocks form)."""
    _check("bonsai_p40_fwht_signs_n", call("bonsai_p40_fwht_signs_n", x, signs, n, stream=stream))


def rmsnorm(x, w, y, n_rows: int, n: int, eps: float, stream=None) -> None:
    _check("bonsai_p40_rmsnorm",
           call("bonsai_p40_rmsnorm", x, w, y, n_rows, n, C.c_float(eps), stream=stream))


def fwht_quant(x, signs, xq, n: int, stream=None) -> None:
    _check("bonsai_p40_fwht_quant", call("bonsai_p40_fwht_quant", x, signs, xq, n, stream=stream))


def quant_tokens(X, signs, Xq, n: int, n_tok: int, rotate: bool, stream=None) -> None:
    _check("bonsai_p40_quant_tokens",
           call("bonsai_p40_quant_tokens", X, signs, Xq, n, n_tok, int(rotate), stream=stream))


def swiglu_fwht_quant(gate, up, signs, xq, n: int, stream=None) -> None:
    _check("bonsai_p40_swiglu_fwht_quant",
           call("bonsai_p40_swiglu_fwht_quant", gate, up, signs, xq, n, stream=stream))


def rmsnorm_fwht_quant(x, w, signs, xq, n: int, n_tok: int, eps: float, stream=None) -> None:
    _check("bonsai_p40_rmsnorm_fwht_quant",
           call("bonsai_p40_rmsnorm_fwht_quant", x, w, signs, xq, n, n_tok, C.c_float(eps),
                stream=stream))


def quant_gemv(W, x, y, n_out: int, n_in: int, stream=None) -> None:
    """y = W . Q8_1(x), one launch (no rotation, no Q8_1 buffer)."""
    _check("bonsai_p40_quant_gemv", call("bonsai_p40_quant_gemv", W, x, y, n_out, n_in, stream=stream))


class GgmlTensor(C.Structure):
    """bonsai_ggml_tensor of include/bonsai_p40_ggml.h: the ggml_tensor fields
    the ggml hook reads."""
    _fields_ = [("type", C.c_int), ("ne", C.c_int64 * 4), ("nb", C.c_size_t * 4), ("data", C.c_void_p)]


GGML_TYPE_F32, GGML_TYPE_PQ2_0 = 0, 142


def ggml_tensor(type_: int, ne, nb, data) -> GgmlTensor:
    """A tensor view: ne and nb of up to 4 dimensions (missing ne are 1, the
    nb of a missing dimension is the size of the one below), data a tensor
    or a device pointer."""
    ne = list(ne) + [1] * (4 - len(ne))
    nb = list(nb)
    while len(nb) < 4:
        nb.append(nb[-1] * ne[len(nb) - 1])
    return GgmlTensor(type_, (C.c_int64 * 4)(*ne), (C.c_size_t * 4)(*nb), _ptr(data))


def ggml_should_use(src0_type: int, device: int, ne11: int) -> bool:
    return lib().bonsai_p40_ggml_should_use(src0_type, device, ne11) == 1


def ggml_mul_mat(src0: GgmlTensor, src1: GgmlTensor, dst: GgmlTensor, scratch=None, scratch_bytes: int = 0,
                 stream=None) -> bool:
    """True when the hook enqueued dst = src0 . src1, False when the caller
    keeps its stock path."""
    return lib().bonsai_p40_ggml_mul_mat(C.byref(src0), C.byref(src1), C.byref(dst), _ptr(scratch),
                                         scratch_bytes, _stream(stream)) == 1


def fwht_gemv(W, x, signs, y, n_out: int, n_in: int, stream=None) -> None:
    _check("bonsai_p40_fwht_gemv",
           call("bonsai_p40_fwht_gemv", W, x, signs, y, n_out, n_in, stream=stream))


def _group_arrays(Ws, ys, n_outs):
    n = len(Ws)
    if not (len(ys) == n and len(n_outs) == n):
        raise ValueError("Ws, ys and n_outs must have the same length")
    Wa = (C.c_void_p * n)(*[_ptr(w) for w in Ws])
    ya = (C.c_void_p * n)(*[_ptr(y) for y in ys])
    na = (C.c_int64 * n)(*[int(r) for r in n_outs])
    # keep the arrays alive for the call: the caller holds the returned tuple
    return (Wa, ya, na), C.cast(Wa, C.c_void_p), C.cast(ya, C.c_void_p), C.cast(na, C.c_void_p), n


def gemv_group(Ws, xq, ys, n_outs, n_in: int, stream=None) -> None:
    """y_m = W_m . xq for up to 4 matrices sharing n_in, one launch."""
    keep, Wp, yp, np_, n = _group_arrays(Ws, ys, n_outs)
    rc = lib().bonsai_p40_gemv_group(Wp, yp, np_, n, _ptr(xq), n_in, _stream(stream))
    del keep
    _check("bonsai_p40_gemv_group", rc)


def fwht_gemv_group(Ws, x, signs, ys, n_outs, n_in: int, stream=None) -> None:
    """y_m = W_m . Q8_1(FWHT(signs .* x)) for up to 4 matrices, one launch."""
    keep, Wp, yp, np_, n = _group_arrays(Ws, ys, n_outs)
    rc = lib().bonsai_p40_fwht_gemv_group(Wp, yp, np_, n, _ptr(x), _ptr(signs), n_in, _stream(stream))
    del keep
    _check("bonsai_p40_fwht_gemv_group", rc)


def rmsnorm_fwht_gemv_group(Ws, x, norm_w, signs, ys, n_outs, n_in: int, eps: float,
                            stream=None) -> None:
    """y_m = W_m . Q8_1(FWHT(signs .* RMSNorm(x, norm_w, eps))), up to 4 matrices, one launch."""
    keep, Wp, yp, np_, n = _group_arrays(Ws, ys, n_outs)
    rc = lib().bonsai_p40_rmsnorm_fwht_gemv_group(Wp, yp, np_, n, _ptr(x), _ptr(norm_w), _ptr(signs), n_in,
                                                  C.c_float(eps), _stream(stream))
    del keep
    _check("bonsai_p40_rmsnorm_fwht_gemv_group", rc)


FFN_SYNC_BYTES = 256


def ffn_workspace_bytes(n_ff: int) -> int:
    """BONSAI_P40_FFN_WORKSPACE_BYTES(n_ff) of include/bonsai_p40.h."""
    return FFN_SYNC_BYTES + 8 * n_ff


def ffn_gate_up_swiglu(Wg, Wu, x, norm_w, x_signs, h_signs, hq, n_ff: int, n_embd: int, eps: float,
                       workspace, status=None, stream=None) -> None:
    """hq = Q8_1(FWHT(h_signs .* swiglu(Wg.a, Wu.a))), a = Q8_1(FWHT(x_signs .*
    RMSNorm(x))) (norm_w None: no RMSNorm), one launch; workspace zero-filled
    before its first use (ffn_workspace_bytes(n_ff) bytes)."""
    _check("bonsai_p40_ffn_gate_up_swiglu",
           call("bonsai_p40_ffn_gate_up_swiglu", Wg, Wu, x, norm_w, x_signs, h_signs, hq, n_ff, n_embd,
                C.c_float(eps), workspace, status, stream=stream))


FFN_NOALLOC_MAX_NFF = 65536


def ffn_gate_up_swiglu_noalloc(Wg, Wu, x, norm_w, x_signs, h_signs, hq, n_ff: int, n_embd: int, eps: float,
                               status=None, stream=None) -> None:
    """ffn_gate_up_swiglu with the library's static per-GPU scratch instead of
    a workspace (n_ff <= FFN_NOALLOC_MAX_NFF; calls on one GPU must not
    overlap)."""
    _check("bonsai_p40_ffn_gate_up_swiglu_noalloc",
           call("bonsai_p40_ffn_gate_up_swiglu_noalloc", Wg, Wu, x, norm_w, x_signs, h_signs, hq, n_ff, n_embd,
                C.c_float(eps), status, stream=stream))


def quantize_pq2_0(x, w, n: int, stream=None) -> None:
    _check("bonsai_p40_quantize_pq2_0", call("bonsai_p40_quantize_pq2_0", x, w, n, stream=stream))


def dequantize_pq2_0(w, y, n: int, stream=None) -> None:
    _check("bonsai_p40_dequantize_pq2_0", call("bonsai_p40_dequantize_pq2_0", w, y, n, stream=stream))


def chunk_dots(W, xq, out, n_out: int, n_in: int, stream=None) -> None:
    _check("bonsai_p40_chunk_dots",
           call("bonsai_p40_chunk_dots", W, xq, out, n_out, n_in, stream=stream))


def reload_tuning() -> None:
    """Re-read the BONSAI_* tuning variables after changing os.environ."""
    _check("bonsai_p40_reload_tuning", lib().bonsai_p40_reload_tuning())


def mfma_probe(kind: int, blocks: int, iters: int, clk, sink, stream=None) -> None:
    _check("bonsai_p40_mfma_probe", call("bonsai_p40_mfma_probe", kind, blocks, iters, clk, sink, stream=stream))


def overlap_probe(mode: int, nf: int, blocks: int, iters: int, sink, stream=None) -> None:
    _check("bonsai_p40_overlap_probe",
           call("bonsai_p40_overlap_probe", mode, nf, blocks, iters, sink, stream=stream))


def launch_probe(blocks: int, threads: int, sink, stream=None) -> None:
    _check("bonsai_p40_launch_probe", call("bonsai_p40_launch_probe", blocks, threads, sink, stream=stream))


def unit_dma_probe(W, n_out: int, n_in: int, sink, stream=None) -> None:
    _check("bonsai_p40_unit_dma_probe", call("bonsai_p40_unit_dma_probe", W, n_out, n_in, sink, stream=stream))


def stream_read(buf, nbytes: int, out, blocks: int, stream=None) -> None:
    _check("bonsai_p40_stream_read",
           call("bonsai_p40_stream_read", buf, nbytes, out, blocks, stream=stream))


# --------------------------------------------------------- sizes / helpers
def pq2_bytes(n_out: int, n_in: int) -> int:
    return n_out * (n_in // QK_PQ2) * PQ2_BYTES


def q8_bytes(n: int, n_tok: int = 1) -> int:
    return n // QK8 * n_tok * Q81_BYTES


# ------------------------------------------------------------ decode chain
CHAIN_Q8, CHAIN_FWHT, CHAIN_RMSNORM_FWHT, CHAIN_SWIGLU = 0, 1, 2, 3
CHAIN_WORKSPACE_BYTES = 4096


class ChainStep(C.Structure):
    """bonsai_p40_chain_step of include/bonsai_p40.h."""
    _fields_ = [("kind", C.c_int), ("n_mat", C.c_int), ("W", C.c_void_p * 4), ("y", C.c_void_p * 4),
                ("n_out", C.c_int64 * 4), ("n_in", C.c_int64), ("x", C.c_void_p), ("x2", C.c_void_p),
                ("norm_w", C.c_void_p), ("signs", C.c_void_p), ("q_out", C.c_void_p), ("eps", C.c_float)]


def chain_step(kind: int, W=(), y=(), n_out=(), n_in: int = 0, x=None, x2=None, norm_w=None, signs=None,
               q_out=None, eps: float = 0.0) -> ChainStep:
    """One step of a decode chain; tensors are kept by pointer (the caller
    keeps them alive while the plan is used)."""
    s = ChainStep()
    s.kind = kind
    s.n_mat = len(W)
    for i, (w, yy, n) in enumerate(zip(W, y, n_out)):
        s.W[i] = _ptr(w)
        s.y[i] = _ptr(yy)
        s.n_out[i] = int(n)
    s.n_in = int(n_in)
    s.x, s.x2, s.norm_w, s.signs, s.q_out = (_ptr(t) for t in (x, x2, norm_w, signs, q_out))
    s.eps = float(eps)
    return s


def chain_plan_bytes(n_steps: int) -> int:
    return int(lib().bonsai_p40_chain_plan_bytes(n_steps))


def chain_plan(steps, plan) -> None:
    """Check the steps and write the device plan into `plan` (a device
    tensor of chain_plan_bytes(len(steps)) bytes).  Blocking."""
    arr = (ChainStep * len(steps))(*steps)
    _check("bonsai_p40_chain_plan", lib().bonsai_p40_chain_plan(C.cast(arr, C.c_void_p), len(steps), _ptr(plan)))


def chain_run(plan, n_steps: int, workspace, status=None, stream=None) -> None:
    _check("bonsai_p40_chain_run",
           call("bonsai_p40_chain_run", plan, n_steps, workspace, status, stream=stream))


class Chain:
    """A planned decode chain with its own plan buffer and workspace."""

    def __init__(self, steps):
        import torch
        self.steps = list(steps)
        self.n = len(self.steps)
        self.plan = torch.empty(chain_plan_bytes(self.n), dtype=torch.uint8, device="cuda")
        self.workspace = torch.zeros(CHAIN_WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        chain_plan(self.steps, self.plan)

    def run(self, stream=None) -> None:
        chain_run(self.plan, self.n, self.workspace, self.status, stream=stream)


# ------------------------------------------------------------ token mixers
F32, F16, BF16, Q8 = 0, 1, 2, 3

_FORMATS = {_V: "P", _I64: "q", C.c_int: "i", C.c_float: "f"}


def _args_struct(name, **fields):
    """The ctypes struct, and pack: its bytes from the fields' values in a row (a third of the time)."""
    types = [(f, t) for t, names in fields["spec"] for f in names.split()]
    return type(name, (C.Structure,), {"_fields_": types, "__doc__": fields["doc"],
                                       "pack": struct.Struct("@" + "".join(_FORMATS[t] for _, t in types) + "0q").pack})


QkNormRopeArgs = _args_struct("QkNormRopeArgs", doc="bonsai_p40_qk_norm_rope_args of include/bonsai_p40.h.", spec=[
    (_V, "q k v"), (_I64, "q_tok q_head q_el k_tok k_head k_el v_tok v_head v_el n_tok"),
    (C.c_int, "n_head n_kv_head head_dim n_rot interleaved"), (C.c_float, "eps"),
    (_V, "q_norm k_norm pos inv_freq slots q_out"), (_I64, "q_out_tok"), (C.c_int, "q_type kv_type"),
    (_V, "k_pages v_pages"), (_I64, "n_pages page_stride"), (C.c_int, "page_size")])
_PAGED = [(_V, "q out"), (_I64, "q_tok out_tok n_tok"), (C.c_int, "n_seq n_head n_kv_head head_dim io_type kv_type"),
          (C.c_float, "scale"), (_V, "k_pages v_pages"), (_I64, "n_pages page_stride"), (C.c_int, "page_size max_pages"),
          (_V, "table"), (_I64, "table_stride"), (_V, "starts kv_len"), (_I64, "max_kv"), (_V, "workspace"),
          (_I64, "workspace_bytes")]
AttnPagedArgs = _args_struct("AttnPagedArgs", doc="bonsai_p40_attn_paged_args of include/bonsai_p40.h.", spec=_PAGED)
AttnSharedArgs = _args_struct("AttnSharedArgs", doc="bonsai_p40_attn_shared_args of include/bonsai_p40.h, the fields of attn in its place.",
                              spec=_PAGED + [(_V, "groups shared"), (_I64, "max_shared"), (C.c_int, "n_group")])
KvReadArgs = _args_struct("KvReadArgs", doc="bonsai_p40_kv_read_args of include/bonsai_p40.h.", spec=[
    (_V, "k_pages v_pages"), (_I64, "n_pages page_stride"), (C.c_int, "page_size n_kv_head head_dim kv_type"), (_V, "slots"),
    (_I64, "n_tok"), (_V, "k_out v_out"), (_I64, "k_tok v_tok"), (C.c_int, "out_type")])
GdnArgs = _args_struct("GdnArgs", doc="bonsai_p40_gdn_args of include/bonsai_p40.h.", spec=[
    (_V, "q k v out"), (_I64, "q_tok k_tok v_tok out_tok"), (_V, "g beta"), (_I64, "gate_tok"),
    (_V, "state state_out"), (_I64, "n_states"), (_V, "slots starts"), (_I64, "n_tok"),
    (C.c_int, "n_seq n_k_head n_v_head k_dim v_dim type tiled"), (C.c_float, "scale l2_eps"), (_I64, "max_new"),
    (_V, "workspace"), (_I64, "workspace_bytes")])

_TYPES = {}


def _types() -> dict:
    if not _TYPES:
        import torch
        _TYPES.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.int32: "int32",
                       torch.int64: "int64", torch.float64: "float64", torch.int8: "int8"})
    return _TYPES


def _type(t) -> int:
    ty = (_TYPES or _types()).get(t.dtype)
    if ty is None or ty.__class__ is str:
        raise ValueError(f"element type {t.dtype}: fp32, f16 or bf16 is wanted")
    return ty


def _flat(t, name: str, dtype, n: int, dev: int) -> int:
    """The address of t, which has n elements of this type, lies in one piece and on device dev."""
    if t.numel() != n or _TYPES.get(t.dtype) != dtype or not t.is_contiguous() or t.get_device() != dev:
        raise ValueError(f"{name}: {n} contiguous {'fp32' if dtype == F32 else dtype} beside q are wanted, "
                         f"not {t.dtype} {tuple(t.shape)} of strides {t.stride()} on {t.device}")
    return t.data_ptr()


def _rows(t, name: str, shape, dev: int) -> int:
    """The token stride of (token, head, element) rows on device dev whose heads follow each other."""
    if t.shape != shape or t.get_device() != dev:
        raise ValueError(f"{name}: shape {tuple(t.shape)} on {t.device}, wanted {tuple(shape)} beside q")
    n, heads, dim = shape
    tok, head, el = t.stride()
    if (el != 1 and dim != 1) or (head != dim and heads != 1):
        raise ValueError(f"{name}: heads have to follow each other, the strides are {t.stride()}")
    return tok if n > 1 else heads * dim          # (one token's stride says nothing)


def _pages(k_pages, v_pages, dev: int):
    """(n_pages, n_kv_head, page_size, head_dim) pages of keys and values: shape, page stride and type."""
    shape, st = k_pages.shape, k_pages.stride()
    vt = v_pages.stride()
    if (len(st) != 4 or v_pages.shape != shape or v_pages.dtype is not k_pages.dtype
            or vt != st and any(a != b and m > 1 for a, b, m in zip(vt, st, shape)) or not dev == k_pages.get_device() == v_pages.get_device()):
        raise ValueError("k_pages and v_pages: alike, (n_pages, n_kv_head, page_size, head_dim), beside q or the outputs")
    n, h, p, d = shape
    page, head, row, el = st
    if (el != 1 and d != 1) or (row != d and p != 1) or (head != p * d and h != 1):
        raise ValueError("a page has to lie in one piece")
    if (_TYPES or _types()).get(k_pages.dtype) != "int8":
        return n, h, p, d, page if n > 1 else h * p * d, _type(k_pages)
    # 8 bits: the scales lie behind the rows of each page, outside the tensor that names these, and a slice of its heads
    # would put them elsewhere: so each tensor's page stride has to be that of its pages.  A view of one page may have
    # lost it ([None] makes it the rows' alone); then its memory has to be this one page and no other
    size = h * p * (d + 4)
    page = size + -size % 16
    for t in (k_pages, v_pages) if n else ():
        at, there = t.storage_offset(), t.untyped_storage().nbytes()
        if n == 1 and t.stride(0) == h * p * d:
            fits = at == 0 and size <= there <= page
        else:
            fits = t.stride(0) == page and at + (n - 1) * page + size <= there
        if not fits:
            raise ValueError("8-bit pages follow each other, each with room for its scales, as q8_pages makes them ([i:i + 1] of these is one page)")
    return n, h, p, d, page, Q8


def q8_pages(n_pages: int, n_kv_head: int, page_size: int, head_dim: int, device="cuda"):
    """Zeroed 8-bit pages (of keys or of values): the whole numbers, int8 (n_pages,
    n_kv_head, page_size, head_dim), which the calls take as k_pages or v_pages, and the
    scales, fp32 (n_pages, n_kv_head, page_size), two views of one piece of memory in
    which a page's scales follow its rows."""
    import torch
    rows, scales = n_kv_head * page_size * head_dim, 4 * n_kv_head * page_size
    page = rows + scales + -(rows + scales) % 16
    memory = torch.zeros((n_pages, page), dtype=torch.int8, device=device)
    # (strided by hand, so that one page, too, has its stride: it tells all heads from some of them)
    return (memory.as_strided((n_pages, n_kv_head, page_size, head_dim), (page, page_size * head_dim, head_dim, 1)),
            memory.view(torch.float32).as_strided((n_pages, n_kv_head, page_size), (page // 4, page_size, 1), rows // 4))


def rope_inv_freq(n_rot: int, base: float, device="cuda"):
    """base^(-2 i / n_rot), i < n_rot / 2, in fp64: the inv_freq of qk_norm_rope."""
    import torch
    return base ** (-torch.arange(0, n_rot, 2, dtype=torch.float64, device=device) / n_rot)


def _scratch(workspace, dev: int):
    if workspace is None:
        return 0, 0
    if workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError("workspace: one piece beside q is wanted")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _stream_of(q, stream) -> int | None:
    """The stream for a call on q's device, which has to be the current one."""
    dev = q.get_device()
    if dev < 0:
        raise ValueError("tensors on the device are wanted")
    if _device is None:
        _init_streams()
    if dev != _device():
        raise ValueError(f"the tensors are on {q.device}, the current device is {_device()}")
    return _raw_stream(dev) if stream is None else _stream(stream)


def _qk_norm_rope_args(q, k, v, q_norm, k_norm, eps, pos, inv_freq, slots, k_pages, v_pages, q_out, interleaved):
    shape, ks, qt = q.shape, k.shape, q.stride()
    if len(qt) != 3 or len(ks) != 3:
        raise ValueError("q, k and v: (n_tok, heads, head_dim) is wanted")
    n, h, d = shape
    nk, kv, dk = ks
    ty = q.dtype
    if _type(q) != F32 or k.dtype is not ty or v.dtype is not ty:
        raise ValueError("q, k and v: fp32 is wanted")
    dev = q.get_device()
    if nk != n or dk != d or v.shape != ks or not dev == k.get_device() == v.get_device():
        raise ValueError(f"k, v: shapes {tuple(ks)}, {tuple(v.shape)} beside q's {tuple(shape)}, on one device")
    pages, page_kv, page_size, page_d, stride, kv_type = _pages(k_pages, v_pages, dev)
    if page_kv != kv or page_d != d:
        raise ValueError("the pages have other heads")
    half = 0 if inv_freq is None else inv_freq.numel()
    return QkNormRopeArgs.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), *qt, *k.stride(), *v.stride(), n, h, kv, d, 2 * half,
        1 if interleaved else 0, eps, 0 if q_norm is None else _flat(q_norm, "q_norm", F32, d, dev),
        0 if k_norm is None else _flat(k_norm, "k_norm", F32, d, dev),
        _flat(pos, "pos", "int32", n, dev) if half else 0, _flat(inv_freq, "inv_freq", "float64", half, dev) if half else 0,
        _flat(slots, "slots", "int64", n, dev), q_out.data_ptr(), _rows(q_out, "q_out", shape, dev), _type(q_out), kv_type,
        k_pages.data_ptr(), v_pages.data_ptr(), pages, stride, page_size)


def qk_norm_rope(q, k, v, q_norm, k_norm, eps: float, pos, inv_freq, slots, k_pages, v_pages, q_out,
                 interleaved: bool = False, stream=None) -> None:
    """RMSNorm of query and key heads (q_norm, k_norm None: none), rotation of
    their first 2 * len(inv_freq) elements, and the append of keys and values to
    the pages.  q, k, v: fp32 (n_tok, heads, head_dim) views with the elements of
    a head or the tokens consecutive (Y.view(heads, head_dim, n_tok).permute(2, 0,
    1) of a gemm)."""
    a = _qk_norm_rope_args(q, k, v, q_norm, k_norm, eps, pos, inv_freq, slots, k_pages, v_pages, q_out, interleaved)
    rc = lib().bonsai_p40_qk_norm_rope(a, _stream_of(q, stream))
    if rc:
        _check("bonsai_p40_qk_norm_rope", rc)


def _attn_args(q, k_pages, v_pages, table, starts, kv_len, out, workspace, max_kv, scale, pack=None, *more):
    shape, entries, steps = q.shape, table.shape, table.stride()
    if len(shape) != 3 or len(steps) != 2:
        raise ValueError("q: (n_tok, heads, head_dim) and table: (n_seq, max_pages) are wanted")
    n, h, d = shape
    io = _type(q)
    if out.dtype is not q.dtype:
        raise ValueError("out has to have q's type")
    dev = q.get_device()
    pages, kv, page_size, page_d, stride, kv_type = _pages(k_pages, v_pages, dev)
    if page_d != d:
        raise ValueError("the pages have another head_dim")
    n_seq, cols = entries
    row, col = steps
    if _TYPES.get(table.dtype) != "int32" or (col != 1 and cols > 1) or table.get_device() != dev:
        raise ValueError("table: int32 rows beside q are wanted")
    ws, ws_bytes = _scratch(workspace, dev)
    return (pack or AttnPagedArgs.pack)(
        q.data_ptr(), out.data_ptr(), _rows(q, "q", shape, dev), _rows(out, "out", shape, dev), n, n_seq, h, kv, d, io, kv_type,
        d ** -0.5 if scale is None else scale, k_pages.data_ptr(), v_pages.data_ptr(), pages, stride, page_size, cols,
        table.data_ptr(), row if n_seq > 1 else cols, _flat(starts, "starts", "int32", n_seq + 1, dev),
        _flat(kv_len, "kv_len", "int32", n_seq, dev), max_kv, ws, ws_bytes, *more)


def attn_paged_workspace_bytes(q, k_pages, v_pages, table, starts, kv_len, out, max_kv: int = 0, scale=None) -> int:
    """bonsai_p40_attn_paged_workspace_bytes for these arguments of attn_paged."""
    a = _attn_args(q, k_pages, v_pages, table, starts, kv_len, out, None, max_kv, scale)
    return int(lib().bonsai_p40_attn_paged_workspace_bytes(a))


def attn_paged(q, k_pages, v_pages, table, starts, kv_len, out, workspace=None, max_kv: int = 0, scale=None,
               stream=None) -> None:
    """Causal attention of every sequence's new tokens (rows starts[s] ..
    starts[s + 1] - 1 of q and out, (n_tok, heads, head_dim)) over its kv_len[s] keys
    in the pages table[s]; scale None: head_dim^-1/2."""
    a = _attn_args(q, k_pages, v_pages, table, starts, kv_len, out, workspace, max_kv, scale)
    rc = lib().bonsai_p40_attn_paged(a, _stream_of(q, stream))
    if rc:
        _check("bonsai_p40_attn_paged", rc)


def _attn_shared_args(q, k_pages, v_pages, table, starts, kv_len, groups, shared, out, workspace, max_kv, max_shared, scale):
    _type(q)
    dev, n = q.get_device(), shared.numel()
    return _attn_args(q, k_pages, v_pages, table, starts, kv_len, out, workspace, max_kv, scale, AttnSharedArgs.pack,
                      _flat(groups, "groups", "int32", n + 1, dev), _flat(shared, "shared", "int32", n, dev), max_shared, n)


def attn_shared_workspace_bytes(q, k_pages, v_pages, table, starts, kv_len, groups, shared, out, max_kv: int = 0,
                                max_shared: int = 0, scale=None) -> int:
    """bonsai_p40_attn_shared_workspace_bytes for these arguments of attn_shared."""
    a = _attn_shared_args(q, k_pages, v_pages, table, starts, kv_len, groups, shared, out, None, max_kv, max_shared, scale)
    return int(lib().bonsai_p40_attn_shared_workspace_bytes(a))


def attn_shared(q, k_pages, v_pages, table, starts, kv_len, groups, shared, out, workspace, max_kv: int = 0,
                max_shared: int = 0, scale=None, stream=None) -> None:
    """attn_paged of a batch whose sequences groups[g] .. groups[g + 1] - 1 begin with
    the same shared[g] keys, those of table[groups[g]], which are read once for all of them.
    max_kv, max_shared: the longest prefix and the most own keys of a sequence together, and that prefix."""
    a = _attn_shared_args(q, k_pages, v_pages, table, starts, kv_len, groups, shared, out, workspace, max_kv, max_shared, scale)
    rc = lib().bonsai_p40_attn_shared(a, _stream_of(q, stream))
    if rc:
        _check("bonsai_p40_attn_shared", rc)


def _kv_read_args(k_pages, v_pages, slots, k_out, v_out):
    shape = k_out.shape
    if len(shape) != 3 or v_out.dtype is not k_out.dtype:
        raise ValueError("k_out and v_out: (n_tok, n_kv_head, head_dim) of one type are wanted")
    n, kv, d = shape
    out, dev = _type(k_out), k_out.get_device()
    pages, page_kv, page_size, page_d, stride, kv_type = _pages(k_pages, v_pages, dev)
    if page_kv != kv or page_d != d:
        raise ValueError("the pages have other heads")
    return KvReadArgs.pack(k_pages.data_ptr(), v_pages.data_ptr(), pages, stride, page_size, kv, d, kv_type,
                           _flat(slots, "slots", "int64", n, dev), n, k_out.data_ptr(), v_out.data_ptr(),
                           _rows(k_out, "k_out", shape, dev), _rows(v_out, "v_out", shape, dev), out)


def kv_read(k_pages, v_pages, slots, k_out, v_out, stream=None) -> None:
    """Rows slots of the pages (16-bit, or 8-bit as q8_pages makes them) into k_out and
    v_out, (n_tok, n_kv_head, head_dim) fp32, f16 or bf16; rows of slots outside stay as they were."""
    a = _kv_read_args(k_pages, v_pages, slots, k_out, v_out)
    rc = lib().bonsai_p40_kv_read(a, _stream_of(k_out, stream))
    if rc:
        _check("bonsai_p40_kv_read", rc)


def _gdn_args(q, k, v, g, beta, state, state_out, out, starts, workspace, max_new, slots, scale, l2_eps, tiled):
    qs, vs, ss, gs = q.shape, v.shape, state.shape, g.stride()
    if len(qs) != 3 or len(vs) != 3 or starts.dim() != 1 or len(ss) != 4 or len(gs) != 2:
        raise ValueError("q, k, v: (n_tok, heads, dim), g, beta: (n_tok, v_heads), state: (n_states, v_heads, k_dim, v_dim) and "
                         "starts: (n_seq + 1,) are wanted")
    n, kh, kd = qs
    nv, vh, vd = vs
    states, sh, sk, sv = ss
    ty, dt = _type(q), q.dtype
    if k.dtype is not dt or v.dtype is not dt or out.dtype is not dt:
        raise ValueError("q, k, v and out: one type is wanted")
    dev = q.get_device()
    if nv != n or sh != vh or sk != kd or sv != vd or state_out.shape != ss:
        raise ValueError(f"v, state, state_out: shapes {tuple(vs)}, {tuple(ss)}, {tuple(state_out.shape)} beside q's {tuple(qs)}")
    if (_type(g) != F32 or beta.dtype is not g.dtype or g.shape != (n, vh) or beta.shape != g.shape
            or not dev == g.get_device() == beta.get_device()):
        raise ValueError(f"g and beta: fp32 ({n}, {vh}) beside q is wanted")
    gt, gh = gs
    bt, bh = beta.stride()
    if (vh > 1 and not gh == bh == 1) or (n > 1 and gt != bt):
        raise ValueError("g and beta: one token stride, and the heads of a token consecutive")
    n_seq, all_states = starts.numel() - 1, states * vh * kd * vd
    ws, ws_bytes = _scratch(workspace, dev)
    return GdnArgs.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _rows(q, "q", qs, dev), _rows(k, "k", qs, dev),
        _rows(v, "v", vs, dev), _rows(out, "out", vs, dev), g.data_ptr(), beta.data_ptr(), gt if n > 1 else vh,
        _flat(state, "state", F32, all_states, dev), _flat(state_out, "state_out", F32, all_states, dev), states,
        0 if slots is None else _flat(slots, "slots", "int32", n_seq, dev),
        _flat(starts, "starts", "int32", n_seq + 1, dev), n, n_seq, kh, vh, kd, vd, ty, 1 if tiled else 0,
        kd ** -0.5 if scale is None else scale, l2_eps, max_new, ws, ws_bytes)


def gdn_workspace_bytes(q, k, v, g, beta, state, state_out, out, starts, max_new: int = 0, slots=None, scale=None,
                        l2_eps: float = 0.0, tiled: bool = False) -> int:
    """bonsai_p40_gdn_workspace_bytes for these arguments of gdn."""
    a = _gdn_args(q, k, v, g, beta, state, state_out, out, starts, None, max_new, slots, scale, l2_eps, tiled)
    return int(lib().bonsai_p40_gdn_workspace_bytes(a))


def gdn(q, k, v, g, beta, state, state_out, out, starts, workspace=None, max_new: int = 0, slots=None, scale=None,
        l2_eps: float = 0.0, tiled: bool = False, stream=None) -> None:
    """The gated delta rule over every sequence's tokens (rows starts[s] ..
    starts[s + 1] - 1): q, k (n_tok, k_heads, k_dim), v, out (n_tok, v_heads, v_dim),
    g (log decay) and beta (n_tok, v_heads), state (n_states, v_heads, k_dim, v_dim);
    scale None: k_dim^-1/2."""
    a = _gdn_args(q, k, v, g, beta, state, state_out, out, starts, workspace, max_new, slots, scale, l2_eps, tiled)
    rc = lib().bonsai_p40_gdn(a, _stream_of(q, stream))
    if rc:
        _check("bonsai_p40_gdn", rc)
