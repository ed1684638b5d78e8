"""Operator-level host interface: torch tensors in, HIP kernels underneath.

``mm8_one`` / ``mm8_three`` / ``wkv_forward`` mirror the reference's native
operators ``torch.ops.rwkv.*`` (reference
src/rwkvstic/agnostic/backends/cuda/wrapper.cpp:45-127): same names, argument
order and in-place semantics.  ``register_torch_ops()`` publishes them under
the same ``rwkv::`` namespace so reference-style modules resolve them.

Every function requires CUDA (ROCm) tensors and raises on anything else;
nothing here falls back to torch arithmetic.
"""
from __future__ import annotations

from contextlib import nullcontext
from typing import Optional, Tuple

import torch

from . import _native as N

_scratch: dict = {}


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _req(t: torch.Tensor, dtype, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def _contig(t: torch.Tensor, name: str) -> None:
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _workspace(nbytes: int, device) -> torch.Tensor:
    """Scratch of one product, from torch's allocator: it belongs to the stream the call runs on, so that calls of other streams
    have others.  A call that is recorded, or runs on another device than its tensors', takes a buffer kept per device: it may be
    replayed at any time, so where a larger one is needed the smaller ones stay (each at least twice the one before)."""
    here = torch.cuda.current_device()
    key = device.index if device.index is not None else here
    if key == here and not torch.cuda.is_current_stream_capturing():
        return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)
    kept = _scratch.setdefault(key, [])
    if not kept or kept[-1].numel() < nbytes:
        kept.append(torch.empty(max(nbytes, 2 * kept[-1].numel() if kept else 1 << 20), dtype=torch.uint8, device=device))
    return kept[-1]


# ---------------------------------------------------------------- reference operators
def _mm8_dtype(x: torch.Tensor, others, what: str) -> torch.dtype:
    """float32 or float64, shared by x, y and r (the dispatch of wrapper.cpp:58-60)."""
    if x.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"{what}: x, y, r must be float32 or float64, got {x.dtype}")
    for t in others:
        _req(t, x.dtype, "x/y/r")
    return x.dtype


def _holds(t: torch.Tensor, n: int) -> bool:
    """Whether the kernels may read or write ``n`` values one after the other from the tensor's first on (a view can have as
    many elements and less memory)."""
    return t.numel() >= n and t.untyped_storage().nbytes() // t.element_size() - t.storage_offset() >= n


def mm8_one(N_in: int, M_out: int, x: torch.Tensor, w: torch.Tensor, y: torch.Tensor, r: torch.Tensor) -> None:
    """``y[k] += sum_j x[j]*(w[j,k]*r[j])``; argument meaning of wrapper.cpp:52-54 (N=in, M=out); x, y, r all
    float32 or all float64 (wrapper.cpp:60-77)."""
    dt = _mm8_dtype(x, (x, y, r), "mm8_one"); _req(w, torch.uint8, "w")
    if x.dim() != 1 or x.stride(0) != 1 or y.stride(0) != 1 or w.dim() != 2 or w.stride(1) != 1:
        raise ValueError("mm8_one: x, y need unit stride and w.stride(1) == 1 (wrapper.cpp:55-57)")
    if not (_holds(x, N_in) and _holds(r, N_in) and _holds(y, M_out)) or w.shape[0] < N_in or w.shape[1] < M_out:
        raise ValueError("mm8_one: tensor smaller than (N, M)")
    L = N.lib()
    f64 = dt == torch.float64
    ws = _workspace((L.rwkv_mm8_f64_workspace_bytes if f64 else L.rwkv_mm8_workspace_bytes)(N_in, M_out, 1), x.device)
    N.check((L.rwkv_mm8_one_f64 if f64 else L.rwkv_mm8_one)(_stream(), N_in, M_out, x.data_ptr(), w.data_ptr(), w.stride(0),
                                                            y.data_ptr(), r.data_ptr(), ws.data_ptr(), ws.numel()))


def mm8_three(N_in: int, M_out: int, x0, x1, x2, w0, w1, w2, y0, y1, y2, r0, r1, r2) -> None:
    """Three ``mm8_one`` problems in one call (wrapper.cpp:82-86); float32 or float64 like ``mm8_one``."""
    dt = _mm8_dtype(x0, (x0, x1, x2, y0, y1, y2, r0, r1, r2), "mm8_three")
    for t in (x0, x1, x2, y0, y1, y2, r0, r1, r2):
        if t.stride(0) != 1:
            raise ValueError("mm8_three: x, y, r need unit stride")
    if not (all(_holds(t, N_in) for t in (x0, x1, x2, r0, r1, r2)) and all(_holds(t, M_out) for t in (y0, y1, y2))):
        raise ValueError("mm8_three: tensor smaller than (N, M)")
    for t in (w0, w1, w2):
        _req(t, torch.uint8, "w")
        if t.dim() != 2 or t.stride(1) != 1 or t.shape[0] < N_in or t.shape[1] < M_out:
            raise ValueError("mm8_three: w must be [>=N, >=M] with unit inner stride")
    L = N.lib()
    f64 = dt == torch.float64
    ws = _workspace((L.rwkv_mm8_f64_workspace_bytes if f64 else L.rwkv_mm8_workspace_bytes)(N_in, M_out, 3), x0.device)
    N.check((L.rwkv_mm8_three_f64 if f64 else L.rwkv_mm8_three)(
        _stream(), N_in, M_out, x0.data_ptr(), x1.data_ptr(), x2.data_ptr(),
        w0.data_ptr(), w0.stride(0), w1.data_ptr(), w1.stride(0), w2.data_ptr(), w2.stride(0),
        y0.data_ptr(), y1.data_ptr(), y2.data_ptr(),
        r0.data_ptr(), r1.data_ptr(), r2.data_ptr(), ws.data_ptr(), ws.numel()))


def wkv_forward(B: int, T: int, C: int, w, u, k, v, y, aa, bb, pp) -> None:
    """float64 WKV with the reference's state convention (wrapper.cpp:45-50)."""
    for name, t in (("w", w), ("u", u), ("k", k), ("v", v), ("y", y), ("aa", aa), ("bb", bb), ("pp", pp)):
        _req(t, torch.float64, name); _contig(t, name)
    if k.numel() < B * T * C or v.numel() < B * T * C or y.numel() < B * T * C:
        raise ValueError("wkv_forward: k/v/y smaller than B*T*C")
    if min(aa.numel(), bb.numel(), pp.numel()) < B * C or min(w.numel(), u.numel()) < C:
        raise ValueError("wkv_forward: state or w/u too small")
    N.check(N.lib().rwkv_wkv_forward_f64(_stream(), B, T, C, w.data_ptr(), u.data_ptr(), k.data_ptr(),
                                         v.data_ptr(), y.data_ptr(), aa.data_ptr(), bb.data_ptr(), pp.data_ptr()))


_registered = False
_SCHEMAS = (
    "wkv_forward(int B, int T, int C, Tensor(a!) w, Tensor(b!) u, Tensor(c!) k, Tensor(d!) v, Tensor(e!) y, Tensor(f!) aa, "
    "Tensor(g!) bb, Tensor(h!) pp) -> ()",
    "mm8_one(int N, int M, Tensor(a!) x, Tensor(b!) w, Tensor(c!) y, Tensor(d!) r) -> ()",
    "mm8_three(int N, int M, Tensor(a!) x, Tensor(b!) x1, Tensor(c!) x2, Tensor(d!) w, Tensor(e!) w1, Tensor(f!) w2, "
    "Tensor(g!) y, Tensor(h!) y1, Tensor(i!) y2, Tensor(j!) r, Tensor(k!) r1, Tensor(l!) r2) -> ()",
)


def register_torch_ops() -> None:
    """Publish ``torch.ops.rwkv.{wkv_forward,mm8_one,mm8_three}`` with the
    reference's schemas (wrapper.cpp:131-141: TORCH_LIBRARY(rwkv, m)).  Their calls run in csrc/rwkv_torch.cpp; what does not
    fit there comes back to the functions above, and all calls do where it is not built."""
    global _registered
    if _registered:
        return
    host = N.host()
    if host is not None:
        host.register_ops(_SCHEMAS)
    else:
        lib = torch.library.Library("rwkv", "DEF")
        for schema in _SCHEMAS:
            lib.define(schema)
        for fn in (wkv_forward, mm8_one, mm8_three):
            lib.impl(fn.__name__, fn, "CUDA")
        register_torch_ops._lib = lib     # keep alive
    _registered = True


# ---------------------------------------------------------------- quantiser / layouts
def _quantize(weight: torch.Tensor, codes: bool, packed: bool, packed16: bool):
    """One quantising pass, its codes written in the layouts asked for (None for the others)."""
    _req(weight, torch.float32, "weight"); _contig(weight, "weight")
    n_out, n_in = weight.shape
    L, dev = N.lib(), weight.device
    c = torch.empty((n_in, n_out), dtype=torch.uint8, device=dev) if codes else None
    p = torch.empty(L.rwkv_packed_bytes(n_in, n_out), dtype=torch.uint8, device=dev) if packed else None
    p16 = torch.empty(L.rwkv_packed_m16_bytes(n_in, n_out), dtype=torch.uint8, device=dev) if packed16 else None
    rng = torch.empty(n_in, dtype=torch.float32, device=dev)
    off = torch.empty(n_in, dtype=torch.float64, device=dev)
    ws = torch.empty(L.rwkv_quantize_workspace_bytes(n_out, n_in), dtype=torch.uint8, device=dev)
    N.check(L.rwkv_quantize_layouts(_stream(), weight.data_ptr(), n_out, n_in, c.data_ptr() if codes else None,
                                    p.data_ptr() if packed else None, p16.data_ptr() if packed16 else None,
                                    rng.data_ptr(), off.data_ptr(), ws.data_ptr(), ws.numel()))
    return c, p, p16, rng, off


def quantize(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``weight[out, in]`` float32 -> ``(codes[in, out] uint8, range[in] float32, offset[in] float64)``
    (MM8.QuantizeMatrix, matmul.py:24-40)."""
    _req(weight, torch.float32, "weight"); _contig(weight, "weight")
    n_out, n_in = weight.shape
    # One launch without a workspace, with the same bits, where it is no slower than three that cut the matrix both ways.  It
    # walks the rows with a workgroup per 64 channels; us of both, 144 / 192 / 208 / 256 rows: of 64 to 8192 channels 18 / 21 / 25 / 28
    # against 20, of 1 channel 16 / 18 / 21 / 23 against 20; 16384 channels 19 / 22 / 25 / 28 against 22 / 23 / 26 / 27; 65536
    # channels 35 / 43 / 49 / 56 against 62 / 65 / 76 / 80.  (64 rows 12 against 18.5.)
    if n_out > max(200, n_in // 64):
        codes, _, _, rng, off = _quantize(weight, True, False, False)
        return codes, rng, off
    codes = torch.empty((n_in, n_out), dtype=torch.uint8, device=weight.device)
    rng = torch.empty(n_in, dtype=torch.float32, device=weight.device)
    off = torch.empty(n_in, dtype=torch.float64, device=weight.device)
    N.check(N.lib().rwkv_quantize_u8(_stream(), weight.data_ptr(), n_out, n_in, codes.data_ptr(), rng.data_ptr(), off.data_ptr()))
    return codes, rng, off


def quantize_packed(weight: torch.Tensor, m16: bool = True):
    """``quantize`` without the intermediate codes: ``(packed, packed16 or None, range, offset)``, the layouts being
    those of ``pack`` and (``m16``) ``pack_m16``."""
    _, packed, packed16, rng, off = _quantize(weight, False, True, m16)
    return packed, packed16, rng, off


def pack(codes: torch.Tensor) -> torch.Tensor:
    """Reference layout ``codes[in, out]`` -> streaming block layout (1-D uint8)."""
    _req(codes, torch.uint8, "codes")
    if codes.dim() != 2 or codes.stride(1) != 1:
        raise ValueError("codes must be 2-D with unit inner stride")
    n_in, n_out = codes.shape
    L = N.lib()
    packed = torch.empty(L.rwkv_packed_bytes(n_in, n_out), dtype=torch.uint8, device=codes.device)
    N.check(L.rwkv_pack_u8(_stream(), codes.data_ptr(), codes.stride(0), n_in, n_out, packed.data_ptr()))
    return packed


def unpack(packed: torch.Tensor, n_in: int, n_out: int) -> torch.Tensor:
    _req(packed, torch.uint8, "packed"); _contig(packed, "packed")
    L = N.lib()
    if packed.numel() < L.rwkv_packed_bytes(n_in, n_out):
        raise ValueError("packed buffer too small")
    codes = torch.empty((n_in, n_out), dtype=torch.uint8, device=packed.device)
    N.check(L.rwkv_unpack_u8(_stream(), packed.data_ptr(), n_in, n_out, codes.data_ptr(), n_out))
    return codes


def pack_m16(codes: torch.Tensor) -> torch.Tensor:
    """Reference layout ``codes[in, out]`` -> 16x64 signed blocks for the matrix-core decode kernel."""
    _req(codes, torch.uint8, "codes")
    if codes.dim() != 2 or codes.stride(1) != 1:
        raise ValueError("codes must be 2-D with unit inner stride")
    n_in, n_out = codes.shape
    L = N.lib()
    packed = torch.empty(L.rwkv_packed_m16_bytes(n_in, n_out), dtype=torch.uint8, device=codes.device)
    N.check(L.rwkv_pack_m16(_stream(), codes.data_ptr(), codes.stride(0), n_in, n_out, packed.data_ptr()))
    return packed


def unpack_m16(packed: torch.Tensor, n_in: int, n_out: int) -> torch.Tensor:
    _req(packed, torch.uint8, "packed"); _contig(packed, "packed")
    L = N.lib()
    if packed.numel() < L.rwkv_packed_m16_bytes(n_in, n_out):
        raise ValueError("packed buffer too small")
    codes = torch.empty((n_in, n_out), dtype=torch.uint8, device=packed.device)
    N.check(L.rwkv_unpack_m16(_stream(), packed.data_ptr(), n_in, n_out, codes.data_ptr(), n_out))
    return codes


def dequant_packed(packed, rng, off, n_in: int, n_out: int) -> torch.Tensor:
    _req(packed, torch.uint8, "packed"); _req(rng, torch.float32, "range"); _req(off, torch.float64, "offset")
    L = N.lib()
    if packed.numel() < L.rwkv_packed_bytes(n_in, n_out) or rng.numel() < n_in or off.numel() < n_in:
        raise ValueError("buffer too small")
    dq = torch.empty((n_in, n_out), dtype=torch.float32, device=packed.device)
    N.check(L.rwkv_dequant_packed(_stream(), packed.data_ptr(), rng.data_ptr(), off.data_ptr(), n_in, n_out,
                                  dq.data_ptr()))
    return dq


# ---------------------------------------------------------------- stand-alone kernels
def _buffer(t: torch.Tensor, dtype, n: int, name: str) -> None:
    """``n`` values that the kernels read or write one after the other."""
    _req(t, dtype, name); _contig(t, name)
    if t.numel() < n:
        raise ValueError(f"{name} too small")


def _matvec_args(x, packed, packed_bytes: int, n_in: int, n_out: int, r_row, m_row, r_col, m_col, out) -> torch.Tensor:
    """Checks what ``mm8_packed`` and ``mm8_m16`` are given; returns the tensor their results go to."""
    _req(x, torch.float32, "x"); _contig(x, "x")
    if x.dim() != 2 or x.shape[1] != n_in:
        raise ValueError("x must be [B, n_in]")
    _buffer(packed, torch.uint8, packed_bytes, "packed weights")
    _buffer(r_row, torch.float32, n_in, "r_row"); _buffer(m_row, torch.float64, n_in, "m_row")
    for t, nm in ((r_col, "r_col"), (m_col, "m_col")):
        if t is not None:
            _buffer(t, torch.float32, n_out, nm)
    y = out if out is not None else torch.empty((x.shape[0], n_out), dtype=torch.float64, device=x.device)
    _buffer(y, torch.float64, x.shape[0] * n_out, "out")
    return y


def mm8_packed(x: torch.Tensor, packed: torch.Tensor, n_in: int, n_out: int,
               r_row: torch.Tensor, m_row: torch.Tensor,
               r_col: Optional[torch.Tensor] = None, m_col: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[B, out]`` float64 for ``x[B, in]`` float32, B in {1, 2, 4, 8}."""
    host = N.host()
    y = host and host.mm8_packed(x, packed, n_in, n_out, r_row, m_row, r_col, m_col, out)
    if y is not None:
        return y
    L = N.lib()
    y = _matvec_args(x, packed, L.rwkv_packed_bytes(n_in, n_out), n_in, n_out, r_row, m_row, r_col, m_col, out)
    B = x.shape[0]
    N.check(L.rwkv_mm8_packed(_stream(), B, n_in, n_out, x.data_ptr(), packed.data_ptr(), r_row.data_ptr(),
                              m_row.data_ptr(), r_col.data_ptr() if r_col is not None else None,
                              m_col.data_ptr() if m_col is not None else None, y.data_ptr()))
    return y


def mm8_m16(x: torch.Tensor, packed16: torch.Tensor, n_in: int, n_out: int,
            r_row: torch.Tensor, m_row: torch.Tensor,
            r_col: Optional[torch.Tensor] = None, m_col: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``mm8_packed`` on the matrix cores: ``y[B, out]`` float64 for ``x[B, in]`` float32, any B in 1..8, weights in
    the M16 layout (``pack_m16``); exact integer sums instead of float32 accumulation."""
    host = N.host()
    y = host and host.mm8_m16(x, packed16, n_in, n_out, r_row, m_row, r_col, m_col, out, workspace)
    if y is not None:
        return y
    L = N.lib()
    y = _matvec_args(x, packed16, L.rwkv_packed_m16_bytes(n_in, n_out), n_in, n_out, r_row, m_row, r_col, m_col, out)
    B = x.shape[0]
    need = L.rwkv_mm8_m16_workspace_bytes(B, n_in)
    ws = workspace if workspace is not None else torch.empty(max(need, 1), dtype=torch.uint8, device=x.device)
    _buffer(ws, ws.dtype, 0, "workspace")               # (its bytes are counted by the library)
    N.check(L.rwkv_mm8_m16(_stream(), B, n_in, n_out, x.data_ptr(), packed16.data_ptr(), r_row.data_ptr(),
                           m_row.data_ptr(), r_col.data_ptr() if r_col is not None else None,
                           m_col.data_ptr() if m_col is not None else None, y.data_ptr(), ws.data_ptr(), ws.numel()))
    return y


def gemm8(x: torch.Tensor, packed16: torch.Tensor, rng: torch.Tensor, off: torch.Tensor,
          n_in: int, n_out: int) -> torch.Tensor:
    """``y[T, n_out] = x[T, n_in] @ dequantised matrix`` with the single-token arithmetic
    (fp32(x*range) as exact fixed point, integer dot products, float64 zero-point term);
    the T > 1 branch of MM8.forward (matmul.py:56-57) without its bfloat16 rounding."""
    _req(x, torch.float64, "x"); _contig(x, "x")
    _req(packed16, torch.uint8, "packed16"); _req(rng, torch.float32, "range"); _req(off, torch.float64, "offset")
    if x.dim() != 2 or x.shape[1] != n_in:
        raise ValueError("gemm8: x must be [T, n_in]")
    T = x.shape[0]
    L = N.lib()
    if packed16.numel() < L.rwkv_packed_m16_bytes(n_in, n_out) or rng.numel() < n_in or off.numel() < n_in:
        raise ValueError("gemm8: matrix buffers smaller than (n_in, n_out)")
    y = torch.empty((T, n_out), dtype=torch.float64, device=x.device)
    ws = _workspace(L.rwkv_gemm8_workspace_bytes(T, n_in, n_out), x.device)
    N.check(L.rwkv_gemm8(_stream(), T, n_in, n_out, x.data_ptr(), packed16.data_ptr(), rng.data_ptr(),
                         off.data_ptr(), y.data_ptr(), ws.data_ptr(), ws.numel()))
    return y


def wkv_f32(w, u, k, v, aa, bb, pp) -> torch.Tensor:
    """Max-shifted float32 WKV; ``k, v`` are ``[B, T, C]``; state ``[B, C]`` updated in place."""
    host = N.host()
    y = host and host.wkv_f32(w, u, k, v, aa, bb, pp)
    if y is not None:
        return y
    for name, t in (("w", w), ("u", u), ("k", k), ("v", v), ("aa", aa), ("bb", bb), ("pp", pp)):
        _req(t, torch.float32, name); _contig(t, name)
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError("k, v must be [B, T, C]")
    B, T, Cn = k.shape
    if min(aa.numel(), bb.numel(), pp.numel()) < B * Cn or min(w.numel(), u.numel()) < Cn:
        raise ValueError("state or w/u too small")
    y = torch.empty_like(k)
    N.check(N.lib().rwkv_wkv_f32(_stream(), B, T, Cn, w.data_ptr(), u.data_ptr(), k.data_ptr(), v.data_ptr(),
                                 y.data_ptr(), aa.data_ptr(), bb.data_ptr(), pp.data_ptr()))
    return y


def sample_token(logits: torch.Tensor, *, greedy: bool = False, temp: float = 1.0, tau: float = 0.8, end_adj: float = 0.0,
                 seed: int = 0, counter: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One choice of the device-side sampler (typical.py:1-17; ``logits[0] += end_adj`` in place first,
    rwkvMaster.py:37); the uniform number is a hash of ``(seed, counter)``."""
    _req(logits, torch.float64, "logits"); _contig(logits, "logits")
    out = out if out is not None else torch.empty(1, dtype=torch.int64, device=logits.device)
    _buffer(out, torch.int64, 1, "out")
    N.check(N.lib().rwkv_sample_token(_stream(), logits.data_ptr(), logits.numel(), 1 if greedy else 0, float(temp),
                                      float(tau), float(end_adj), int(seed) & (2 ** 64 - 1), int(counter), out.data_ptr()))
    return out


def argmax(logits: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    _req(logits, torch.float64, "logits"); _contig(logits, "logits")
    out = out if out is not None else torch.empty(1, dtype=torch.int64, device=logits.device)
    _buffer(out, torch.int64, 1, "out")
    N.check(N.lib().rwkv_argmax_f64(_stream(), logits.data_ptr(), logits.numel(), out.data_ptr()))
    return out


# ---------------------------------------------------------------- operators of a serving step over the rows of many requests
_TYPES = {torch.float32: 0, torch.float64: 1, torch.bfloat16: 2, torch.float16: 3}         # rwkv_type


def _is(t, dtypes, shape, name: str, device=None) -> None:
    """A CUDA tensor of one of these types and of this shape, on ``device``."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(map(str, dtypes))}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}")


def _elsewhere(t: torch.Tensor):
    """The device of ``t``, made the current one, where it is another: a launch goes to the current device."""
    return torch.cuda.device(t.device) if t.device.type == "cuda" and t.device.index != torch.cuda.current_device() else None


def _rows(t: torch.Tensor, name: str) -> int:
    """The distance of the rows of ``t [T, ...]``, each of them contiguous."""
    if t.numel() and not t[0].is_contiguous():
        raise ValueError(f"{name} must have contiguous rows")
    return t.stride(0) if t.shape[0] > 1 else t[0].numel() if t.shape[0] else 0


def _apart(t: torch.Tensor, name: str) -> None:
    """Rows that are written must not share memory."""
    if t.shape[0] > 1 and t.stride(0) < t[0].numel():
        raise ValueError(f"{name} must not have rows that overlap")


def lora_rows(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapter: torch.Tensor, scale: Optional[torch.Tensor] = None,
              base: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Low-rank adapters of many requests beside a projection that they share (``gemm8``, ``mm8_m16``):
    ``out[t] = base[t] + scale[i] * b[i] @ (a[i] @ x[t])`` with ``i = adapter[t]``.

    ``x [T, n_in]`` and ``base [T, n_out]`` float32 or float64 (products and sums are computed in that type), ``a [N, R, n_in]``
    and ``b [N, n_out, R]`` bfloat16, float16 or float32 with ``R <= 256`` (adapters of smaller rank are filled up with zeros),
    ``adapter [T]`` int32: a row whose number is outside ``0..N-1`` has no adapter and gets ``base[t]``
    (``N`` may be 0).  ``scale [N]`` float32;
    without it 1.  ``base``: the shared projection's result, without it 0.  ``out`` may be ``base`` itself and may lie
    over ``x``; otherwise it shares no memory with what is read."""
    host = N.host()
    y = host and host.lora_rows(x, a, b, adapter, scale, base, out)
    if y is not None:
        return y
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or not isinstance(a, torch.Tensor) or a.dim() != 3 or not isinstance(b, torch.Tensor) or b.dim() != 3:
        raise ValueError("lora_rows: x must be [T, n_in], a [N, R, n_in], b [N, n_out, R]")
    (T, n_in), (n, R, _), n_out, dev = x.shape, a.shape, b.shape[1], x.device
    _is(x, (torch.float32, torch.float64), (T, n_in), "x")
    _is(a, (torch.bfloat16, torch.float16, torch.float32), (n, R, n_in), "a", dev); _contig(a, "a")
    _is(b, (a.dtype,), (n, n_out, R), "b", dev); _contig(b, "b")
    _is(adapter, (torch.int32,), (T,), "adapter", dev); _contig(adapter, "adapter")
    if scale is not None:
        _is(scale, (torch.float32,), (n,), "scale", dev); _contig(scale, "scale")
    if base is not None:
        _is(base, (x.dtype,), (T, n_out), "base", dev)
    out = torch.empty((T, n_out), dtype=x.dtype, device=dev) if out is None else out
    _is(out, (x.dtype,), (T, n_out), "out", dev); _apart(out, "out")
    strides = _rows(x, "x"), _rows(base, "base") if base is not None else 0, _rows(out, "out")
    if T == 0:
        return out
    L, real = N.lib(), _TYPES[x.dtype]
    with _elsewhere(x) or nullcontext():
        ws = torch.empty(L.rwkv_lora_rows_workspace_bytes(T, n_in, n_out, n, R, real), dtype=torch.uint8, device=dev)
        N.check(L.rwkv_lora_rows(_stream(), T, n_in, n_out, n, R, real, x.data_ptr(), strides[0], _TYPES[a.dtype], a.data_ptr(), b.data_ptr(),
                                 adapter.data_ptr(), scale.data_ptr() if scale is not None else None,
                                 base.data_ptr() if base is not None else None, strides[1], out.data_ptr(), strides[2], ws.data_ptr(), ws.numel()))
    return out


def _default_scale(q) -> float:
    return q.shape[-1] ** -0.5 if isinstance(q, torch.Tensor) and q.dim() and q.shape[-1] else 1.0


def delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, state: torch.Tensor,
               starts: Optional[torch.Tensor] = None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The gated delta rule over packed sequences.  Per value head, row by row, with a state ``S [dk, dv]``:
    ``S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q``.

    ``q, k [T, Hk, dk]`` and ``v [T, Hv, dv]`` float32, bfloat16 or float16 (rows may be apart, heads are contiguous; ``dk <= 256``),
    value head ``h`` with key head ``h // (Hv // Hk)``; ``g`` (logarithm of the decay, at most 0) and ``beta [T, Hv]`` float32;
    ``state [B, Hv, dk, dv]`` float32, updated in place.  ``starts [B + 1]`` int32 on the device: sequence ``b`` is the rows
    ``starts[b]`` to ``starts[b + 1] - 1``; without it ``T / B`` rows each.  ``scale``: ``dk ** -0.5`` unless given.
    Returns ``o [T, Hv, dv]`` of v's type (``out``, which shares no memory with the arguments); rows of no sequence are not written,
    and an empty sequence keeps its state.  From 48 rows a sequence on, on average, chunks of 64 rows are computed at once: a value in them
    that is not finite reaches rows of the chunk before it too, though no other sequence, and keys with ``beta k.k`` over 2 may overflow
    where single steps do not."""
    scale = None if scale is None else float(scale)
    host = N.host()
    y = host and host.delta_rule(q, k, v, g, beta, state, starts, scale if scale is not None else _default_scale(q), out)
    if y is not None:
        return y
    for t, name in ((q, "q"), (v, "v")):
        if not isinstance(t, torch.Tensor) or t.dim() != 3:
            raise ValueError(f"delta_rule: {name} must be [T, heads, channels]")
    if not isinstance(state, torch.Tensor) or state.dim() != 4:
        raise ValueError("delta_rule: state must be [B, Hv, dk, dv]")
    (T, Hk, dk), (_, Hv, dv), B, dev = q.shape, v.shape, state.shape[0], q.device
    _is(q, (torch.float32, torch.bfloat16, torch.float16), (T, Hk, dk), "q")
    _is(k, (q.dtype,), (T, Hk, dk), "k", dev); _is(v, (q.dtype,), (T, Hv, dv), "v", dev)
    for t, name in ((g, "g"), (beta, "beta")):
        _is(t, (torch.float32,), (T, Hv), name, dev); _contig(t, name)
    _is(state, (torch.float32,), (B, Hv, dk, dv), "state", dev); _contig(state, "state")
    if starts is not None:
        _is(starts, (torch.int32,), (B + 1,), "starts", dev); _contig(starts, "starts")
    elif B and T % B:
        raise ValueError("delta_rule: without starts T must be a multiple of the sequences")
    out = torch.empty((T, Hv, dv), dtype=q.dtype, device=dev) if out is None else out
    _is(out, (q.dtype,), (T, Hv, dv), "out", dev); _contig(out, "out")
    strides = _rows(q, "q"), _rows(k, "k"), _rows(v, "v")
    if T == 0 or B == 0:
        return out
    L = N.lib()
    with _elsewhere(q) or nullcontext():
        ws = torch.empty(L.rwkv_delta_rule_workspace_bytes(T, B, Hk, Hv, dk, dv), dtype=torch.uint8, device=dev)
        N.check(L.rwkv_delta_rule(_stream(), T, B, Hk, Hv, dk, dv, _TYPES[q.dtype], q.data_ptr(), strides[0], k.data_ptr(), strides[1], v.data_ptr(),
                                  strides[2], g.data_ptr(), beta.data_ptr(), scale if scale is not None else _default_scale(q),
                                  starts.data_ptr() if starts is not None else None, state.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel()))
    return out


def verify_drafts(logits: torch.Tensor, drafts: torch.Tensor, u: Optional[torch.Tensor] = None, *, draft_logits: Optional[torch.Tensor] = None,
                  lengths: Optional[torch.Tensor] = None, temp: float = 1.0, greedy: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Drafted tokens held against the target's distribution (speculative sampling); returns ``(tokens [B, K+1], accepted [B])`` int64.

    ``logits [B, K+1, V]`` float64 or float32: row ``i`` is the target's for the place of draft ``i`` (the logits after the token before
    it), the last one for the token after all drafts; ``drafts [B, K]`` int64, of which the first ``lengths[b]`` (int32) count.  With
    ``p = softmax(logits / temp)`` and ``q = softmax(draft_logits / temp)`` draft ``d`` is accepted while ``u[b, i] q(d) < p(d)``; at the
    first refused one a token is drawn from ``max(p - q, 0)``, after the last from ``p``, by ``u[b, K]`` (``u [B, K+1]`` float32 in [0, 1)):
    the lowest index at which the running weight exceeds ``u`` times the whole.  ``draft_logits [B, K, V]`` of logits' type; without them
    the drafts have no distribution of their own (``q(d) = 1``).  ``greedy``: a draft is accepted while it is the first maximum, and the
    token drawn is that maximum.  Logits of -infinity are left out: a sampler that keeps only some of the tokens (``sample_token`` does, as
    ``typical``) is verified against once the others are set to that.  Row ``b`` of ``tokens`` is the accepted drafts, the token drawn, then -1 (there too, where no logit has weight)."""
    temp, greedy = float(temp), bool(greedy)
    host = N.host()
    y = host and host.verify_drafts(logits, drafts, u, draft_logits, lengths, temp, greedy)
    if y is not None:
        return y
    if not isinstance(logits, torch.Tensor) or logits.dim() != 3 or logits.shape[1] < 1:
        raise ValueError("verify_drafts: logits must be [B, K + 1, V]")
    (B, K1, V), dev = logits.shape, logits.device
    _is(logits, (torch.float64, torch.float32), logits.shape, "logits")
    _is(drafts, (torch.int64,), (B, K1 - 1), "drafts", dev); _contig(drafts, "drafts")
    if draft_logits is not None:
        _is(draft_logits, (logits.dtype,), (B, K1 - 1, V), "draft_logits", dev)
    for t, name in ((logits, "logits"), (draft_logits, "draft_logits")):
        if t is not None and t.numel() and t.stride(2) != 1 and V > 1:
            raise ValueError(f"{name} must have contiguous rows")
    if lengths is not None:
        _is(lengths, (torch.int32,), (B,), "lengths", dev); _contig(lengths, "lengths")
    if u is not None:
        _is(u, (torch.float32,), (B, K1), "u", dev); _contig(u, "u")
    elif not greedy:
        raise ValueError("verify_drafts: u is needed unless greedy")
    if not greedy and not temp > 0:
        raise ValueError("verify_drafts: temp must be positive")
    tokens, accepted = torch.empty((B, K1), dtype=torch.int64, device=dev), torch.empty(B, dtype=torch.int64, device=dev)
    if B == 0:
        return tokens, accepted
    L = N.lib()
    opt = lambda t: t.data_ptr() if t is not None else None
    by = draft_logits.stride() if draft_logits is not None else (0, 0)
    with _elsewhere(logits) or nullcontext():
        ws = torch.empty(L.rwkv_verify_drafts_workspace_bytes(B, K1 - 1, V), dtype=torch.uint8, device=dev)
        N.check(L.rwkv_verify_drafts(_stream(), B, K1 - 1, V, _TYPES[logits.dtype], logits.data_ptr(), logits.stride(0), logits.stride(1),
                                     opt(draft_logits), by[0], by[1], drafts.data_ptr(), opt(lengths), opt(u), temp, 1 if greedy else 0,
                                     tokens.data_ptr(), accepted.data_ptr(), ws.data_ptr(), ws.numel()))
    return tokens, accepted
