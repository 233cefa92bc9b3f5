"""CudaOps: the reference's MetalOps operator vocabulary
(src/u15-metal-ops.h:59-403 of the reference) over libu15c's C ABI.

Method names, argument meaning and order follow MetalOps; where MetalOps
takes an encoder, these take the current torch CUDA stream; buffers are
torch CUDA tensors (bf16 unless named otherwise) standing in for
SharedBuffers. Errors raise U15Error (the reference returns bool + err).
torch supplies device memory and streams only; every computation runs in
libu15c's kernels.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from ._lib import check, lib


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream():
    # the raw handle: 0.2 us, where building torch.cuda.current_stream() took 3.3 us,
    # as long as the launch itself
    return _raw_stream(torch.cuda.current_device())


def _public_stream(device):
    return torch.cuda.current_stream(device).cuda_stream


# torch's own bindings, where this build of it has them (one without CUDA does not)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_stream)
# the current device, for calls that hold CUDA tensors
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


# array types, kept: making one takes longer than filling it
_INTS = [C.c_int * n for n in range(10)]


def segments_arrays(segments, rows):
    """[(start, end, expert), ...] -> (off int[n+1], expert int[n], n); None, None, 0
    where one segment of expert 0 covers all rows (the ABI's default)."""
    if not segments:
        return None, None, 0
    n = len(segments)
    if n == 1 and segments[0] == (0, rows, 0):
        return None, None, 0   # one segment of expert 0: what no segments stand for
    t_off, t_ex = (_INTS[n + 1], _INTS[n]) if n < 9 else (C.c_int * (n + 1), C.c_int * n)
    return t_off(*[s[0] for s in segments], segments[-1][1]), t_ex(*[s[2] for s in segments]), n


def _bf16(t):
    if t.dtype != torch.bfloat16 or not t.is_cuda or not t.is_contiguous():
        raise L.U15Error(L.EINVAL, "expected a contiguous CUDA bf16 tensor")
    return t


_E4M3 = (torch.uint8, torch.float8_e4m3fn)
_BF16 = (torch.bfloat16,)
_F32 = (torch.float32,)
_BYTES = (torch.uint8,)


def _need(dev, what, t, n, dtypes):
    """The address of `t`, which must hold at least `n` values of one of `dtypes`,
    contiguous on device `dev` (the current one)."""
    if (t is None or t.numel() < n or t.dtype not in dtypes or t.get_device() != dev
            or not t.is_contiguous()):
        raise L.U15Error(L.EINVAL, f"{what}: expected {n} contiguous values of "
                         f"{' or '.join(str(d) for d in dtypes)} on the current device")
    return t.data_ptr()


def _experts(what, t):
    """How many matrices the stack `t` holds."""
    if t is None or t.dim() == 0:
        raise L.U15Error(L.EINVAL, f"{what}: expected a stack of every expert's tensor")
    return t.shape[0]


def _need_scale(dev, what, t, rows, cols, n_experts=1):
    """The same for the packed scales of a quantised [n_experts][rows][cols]."""
    return _need(dev, what, t, n_experts * ((rows + 127) // 128) * ((cols + 511) // 512) * 512,
                 _BYTES)


class CudaOps:
    """MetalOps mirror. One instance per device; stateless apart from that."""

    def __init__(self, device: int = 0):
        self.device = device
        check(lib().u15c_init(device, 0))

    # ---- GEMMs -------------------------------------------------------
    def linear(self, x, w, bias, y, M, K, N):
        check(lib().u15c_linear_bf16(_stream(), _p(_bf16(x)), _p(_bf16(w)), _p(bias), _p(y),
                                     M, K, N))

    def mot_linear(self, x, w_stack, segments, y, M, K, N, epilogue=L.EPI_STORE, bias=None,
                   resid=None):
        off, ex, n = segments_arrays(segments, M)
        check(lib().u15c_mot_linear_bf16(_stream(), _p(x), _p(w_stack), w_stack.shape[0], off,
                                         ex, n, epilogue, _p(bias), _p(resid), _p(y), M, K, N))

    def quant_rows_i8(self, x, q, scale, rows, cols):
        check(lib().u15c_quant_rows_i8(_stream(), _p(x), _p(q), _p(scale), rows, cols))

    def linear_i8(self, xq, s_tok, wq, s_ch, y, M, K, N, bias=None, acc_dump=None):
        check(lib().u15c_linear_i8(_stream(), _p(xq), _p(s_tok), _p(wq), _p(s_ch), _p(bias),
                                   _p(y), _p(acc_dump), M, K, N))

    def mot_linear_i8(self, xq, s_tok, wq_stack, s_ch_stack, segments, y, M, K, N,
                      epilogue=L.EPI_STORE, resid=None, acc_dump=None):
        off, ex, n = segments_arrays(segments, M)
        check(lib().u15c_mot_linear_i8(_stream(), _p(xq), _p(s_tok), _p(wq_stack),
                                       _p(s_ch_stack), wq_stack.shape[0], off, ex, n, epilogue,
                                       _p(resid), _p(y), _p(acc_dump), M, K, N))

    # ---- norms, rope, layout -----------------------------------------
    def rms_norm(self, x, w, y, rows, dim, eps):
        check(lib().u15c_rms_norm(_stream(), _p(x), _p(w), _p(y), rows, dim, eps))

    def mot_rms_norm(self, x, w_stack, segments, y, rows, dim, eps):
        off, ex, n = segments_arrays(segments, rows)
        check(lib().u15c_mot_rms_norm(_stream(), _p(x), _p(w_stack), w_stack.shape[0], off, ex,
                                      n, _p(y), rows, dim, eps))

    def mot_rms_norm_quant_i8(self, x, w_stack, segments, q, scale, rows, dim, eps):
        off, ex, n = segments_arrays(segments, rows)
        check(lib().u15c_mot_rms_norm_quant_i8(_stream(), _p(x), _p(w_stack), w_stack.shape[0],
                                               off, ex, n, _p(q), _p(scale), rows, dim, eps))

    def split_qk_norm(self, x, w_t, w_hw, heads, tokens, head_dim, eps):
        check(lib().u15c_split_qk_norm(_stream(), _p(x), _p(w_t), _p(w_hw), heads, tokens,
                                       head_dim, eps))

    def split_rope(self, x, cos, sin, heads, tokens, head_dim, d_t, d_h):
        check(lib().u15c_split_rope(_stream(), _p(x), _p(cos), _p(sin), heads, tokens,
                                    head_dim, d_t, d_h))

    def build_rope_tables(self, pos_t, pos_h, pos_w, head_dim=128, d_t=64, d_h=32,
                          theta_t=5e6, theta_hw=1e4):
        """Returns (cos, sin) f32 [T][head_dim]; positions are int32 CUDA tensors."""
        T = pos_t.numel()
        c = torch.empty(T, head_dim, dtype=torch.float32, device=pos_t.device)
        s = torch.empty_like(c)
        check(lib().u15c_build_rope_tables(_stream(), _p(pos_t), _p(pos_h), _p(pos_w), T,
                                           head_dim, d_t, d_h, theta_t, theta_hw, _p(c), _p(s)))
        return c, s

    def qkv_post(self, qkv, norms_stack, segments, cos, sin, q_out, k_cache, v_cache,
                 page_table, cap, heads, kv_heads, T, kv_off, eps):
        off, ex, n = segments_arrays(segments, T)
        check(lib().u15c_qkv_post(_stream(), _p(qkv), _p(norms_stack), norms_stack.shape[0],
                                  off, ex, n, _p(cos), _p(sin), _p(q_out), _p(k_cache),
                                  _p(v_cache), _p(page_table), cap, heads, kv_heads, T, kv_off,
                                  eps))

    def transpose_thd(self, x, out, T, H, D):
        check(lib().u15c_transpose_thd(_stream(), _p(x), _p(out), T, H, D))

    def transpose_htd(self, x, out, T, H, D):
        check(lib().u15c_transpose_htd(_stream(), _p(x), _p(out), T, H, D))

    def transpose_into_cache(self, x, cache, T, H, D, cap, offset):
        check(lib().u15c_transpose_into_cache(_stream(), _p(x), _p(cache), T, H, D, cap,
                                              offset))

    def kv_append(self, x, pages, page_table, T, H, offset):
        check(lib().u15c_kv_append(_stream(), _p(x), _p(pages), _p(page_table), T, H, offset))

    # ---- 8-bit floating point, one scale per block of 128 -------------
    # q buffers are uint8 or float8_e4m3fn; scale buffers uint8, packed
    # (include/u15c.h); every tensor is checked for type, size and device.
    def fp8_scale(self, rows, cols, n_experts=1, device="cuda"):
        """Packed scale bytes for a quantised [n_experts][rows][cols]."""
        n = n_experts * lib().u15c_fp8_scale_bytes(rows, cols)
        return torch.empty(n, dtype=torch.uint8, device=device)

    def quant_rows_fp8(self, x, q, scale, rows, cols):
        n, d = rows * cols, _device()
        check(lib().u15c_quant_rows_fp8(_raw_stream(d), _need(d, "x", x, n, _BF16),
                                        _need(d, "q", q, n, _E4M3),
                                        _need_scale(d, "scale", scale, rows, cols), rows, cols))

    def quant_weight_fp8(self, w, q, scale, n_experts, N, K):
        n, d = n_experts * N * K, _device()
        check(lib().u15c_quant_weight_fp8(_raw_stream(d), _need(d, "w", w, n, _BF16),
                                          _need(d, "q", q, n, _E4M3),
                                          _need_scale(d, "scale", scale, N, K, n_experts),
                                          n_experts, N, K))

    def dequant_fp8(self, q, scale, y, rows, cols, n_experts=1):
        n, d = n_experts * rows * cols, _device()
        check(lib().u15c_dequant_fp8(_raw_stream(d), _need(d, "q", q, n, _E4M3),
                                     _need_scale(d, "scale", scale, rows, cols, n_experts),
                                     _need(d, "y", y, n, _BF16), n_experts, rows, cols))

    def mot_add_rms_norm_quant_fp8(self, x, delta, w_stack, segments, x_out, q, scale, rows, dim,
                                   eps):
        off, ex, ns = segments_arrays(segments, rows)
        n, d, E = rows * dim, _device(), _experts("w_stack", w_stack)
        check(lib().u15c_mot_add_rms_norm_quant_fp8(
            _raw_stream(d), _need(d, "x", x, n, _BF16),
            None if delta is None else _need(d, "delta", delta, n, _BF16),
            _need(d, "w_stack", w_stack, E * dim, _BF16), E, off, ex, ns,
            None if x_out is None else _need(d, "x_out", x_out, n, _BF16),
            _need(d, "q", q, n, _E4M3), _need_scale(d, "scale", scale, rows, dim), rows, dim,
            eps))

    def mot_linear_fp8(self, xq, sx, wq_stack, sw_stack, segments, y, M, K, N,
                       epilogue=L.EPI_STORE, resid=None, bias=None):
        off, ex, ns = segments_arrays(segments, M)
        d, E = _device(), _experts("wq_stack", wq_stack)
        ny = M * (N // 2 if epilogue == L.EPI_SWIGLU else N)
        check(lib().u15c_mot_linear_fp8(
            _raw_stream(d), _need(d, "xq", xq, M * K, _E4M3), _need_scale(d, "sx", sx, M, K),
            _need(d, "wq_stack", wq_stack, E * N * K, _E4M3),
            _need_scale(d, "sw_stack", sw_stack, N, K, E), E, off, ex, ns, epilogue,
            None if bias is None else _need(d, "bias", bias, E * N, _BF16),
            None if resid is None else _need(d, "resid", resid, M * N, _BF16),
            _need(d, "y", y, ny, _F32 if epilogue == L.EPI_STORE_F32 else _BF16), M, K, N))

    def mot_swiglu_fp8(self, xq, sx, wq_stack, sw_stack, segments, yq, sy, M, K, N):
        off, ex, ns = segments_arrays(segments, M)
        d, E = _device(), _experts("wq_stack", wq_stack)
        check(lib().u15c_mot_swiglu_fp8(
            _raw_stream(d), _need(d, "xq", xq, M * K, _E4M3), _need_scale(d, "sx", sx, M, K),
            _need(d, "wq_stack", wq_stack, E * N * K, _E4M3),
            _need_scale(d, "sw_stack", sw_stack, N, K, E), E, off, ex, ns,
            _need(d, "yq", yq, M * (N // 2), _E4M3), _need_scale(d, "sy", sy, M, N // 2), M, K,
            N))

    def ffn_fp8_workspace(self, rows, hidden, inter, device="cuda"):
        n = lib().u15c_ffn_fp8_workspace_bytes(rows, hidden, inter)
        return torch.empty(n, dtype=torch.uint8, device=device)

    def mot_ffn_fp8(self, x, delta, w_norm_stack, gu, gu_scale, down, down_scale, segments, y, ws,
                    rows, hidden, inter, eps):
        off, ex, ns = segments_arrays(segments, rows)
        d, E, n = _device(), _experts("gu", gu), rows * hidden
        ws_n = lib().u15c_ffn_fp8_workspace_bytes(rows, hidden, inter)
        check(lib().u15c_mot_ffn_fp8(
            _raw_stream(d), _need(d, "x", x, n, _BF16),
            None if delta is None else _need(d, "delta", delta, n, _BF16),
            _need(d, "w_norm_stack", w_norm_stack, E * hidden, _BF16),
            _need(d, "gu", gu, E * 2 * inter * hidden, _E4M3),
            _need_scale(d, "gu_scale", gu_scale, 2 * inter, hidden, E),
            _need(d, "down", down, E * hidden * inter, _E4M3),
            _need_scale(d, "down_scale", down_scale, hidden, inter, E), E, off, ex, ns,
            _need(d, "y", y, n, _BF16), _need(d, "ws", ws, ws_n, _BYTES), rows, hidden, inter,
            eps))

    # ---- elementwise -------------------------------------------------
    def swiglu(self, gate, up, y, rows, inter):
        check(lib().u15c_swiglu(_stream(), _p(gate), _p(up), _p(y), rows, inter))

    def add(self, dst, src, n):
        check(lib().u15c_add(_stream(), _p(dst), _p(src), n))

    def add_row(self, dst, row, rows, dim):
        check(lib().u15c_add_row(_stream(), _p(dst), _p(row), rows, dim))

    def silu(self, x, n):
        check(lib().u15c_silu(_stream(), _p(x), n))

    # ---- attention ---------------------------------------------------
    def sage_workspace(self, hq, hkv, tq, tk, device="cuda"):
        n = lib().u15c_sage_workspace_bytes(hq, hkv, tq, tk)
        return torch.empty(n, dtype=torch.uint8, device=device)

    def attention(self, q, k, v, out, hq, hkv, tq, tk, cap=0, page_table=None,
                  mode=L.ATTN_BIDIRECTIONAL, q_offset=0, t_index=None, sage_ws=None):
        check(lib().u15c_attention(_stream(), _p(q), _p(k), _p(v), _p(page_table), cap, _p(out),
                                   hq, hkv, tq, tk, 128, mode, q_offset, _p(t_index),
                                   _p(sage_ws)))

    def attention_paged(self, q, k_pages, vt_pages, out, hq, hkv, tq, tk, page_table=None,
                        n_pages=None, mode=L.ATTN_BIDIRECTIONAL, q_offset=0, t_index=None,
                        sage_ws=None):
        """The model's cache layout: K pages [P][hkv][64][128], V pages transposed
        [P][hkv][128][64]; bidirectional runs the tcgen05 kernel."""
        n_pages = k_pages.shape[0] if n_pages is None else n_pages
        check(lib().u15c_attention_paged(_stream(), _p(q), _p(k_pages), _p(vt_pages),
                                         _p(page_table), n_pages, _p(out), hq, hkv, tq, tk, 128,
                                         mode, q_offset, _p(t_index), _p(sage_ws)))

    def sdpa(self, q, k, v, out, hq, hkv, tq, tk, d, cap, causal, q_offset=0):
        check(lib().u15c_sdpa(_stream(), _p(q), _p(k), _p(v), _p(out), hq, hkv, tq, tk, d, cap,
                              int(causal), q_offset))

    def sdpa_steel(self, q, k, v, out, hq, hkv, tq, tk, d, cap, sage_ws=None):
        check(lib().u15c_sdpa_steel(_stream(), _p(q), _p(k), _p(v), _p(out), hq, hkv, tq, tk, d,
                                    cap, _p(sage_ws)))

    def sdpa_block_causal(self, q, k, v, out, t_index, hq, hkv, tq, tk, d, cap, q_offset):
        check(lib().u15c_sdpa_block_causal(_stream(), _p(q), _p(k), _p(v), _p(out),
                                           _p(t_index), hq, hkv, tq, tk, d, cap, q_offset))

    # ---- status ------------------------------------------------------
    def sync(self):
        check(lib().u15c_sync(_stream()))

    def device_status(self) -> int:
        code = C.c_uint(0)
        check(lib().u15c_device_status(self.device, C.byref(code)))
        return code.value
