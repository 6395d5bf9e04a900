"""Typed wrappers over the libmlkb200 C ABI.

Device buffers are passed as torch CUDA tensors (torch provides device memory
and streams only); every computation happens in libmlkb200.so. Host buffers
are numpy arrays or CPU tensors.
"""
from __future__ import annotations

import ctypes as C
from typing import Sequence

import numpy as np

from . import BF16, F16, F32, F64, check, kir, lib

ASSEMBLE_DEVICE0 = 1  # MLKB_ASSEMBLE_DEVICE0
ASSEMBLE_VIA_NCCL = 2  # MLKB_ASSEMBLE_VIA_NCCL

_TORCH_DT = None


def _dt_of(x) -> int:
    global _TORCH_DT
    if isinstance(x, np.ndarray):
        return {np.dtype(np.float16): F16, np.dtype(np.float32): F32,
                np.dtype(np.float64): F64}[x.dtype]
    if _TORCH_DT is None:
        import torch

        _TORCH_DT = {torch.float16: F16, torch.float32: F32, torch.float64: F64}
    return _TORCH_DT[x.dtype]


def _ptr(x) -> int:
    if x is None:
        return None
    if isinstance(x, np.ndarray):
        if not x.flags["C_CONTIGUOUS"]:
            raise ValueError("host buffers must be C-contiguous")
        return x.ctypes.data
    if not x.is_contiguous():
        raise ValueError("tensors must be contiguous")
    return x.data_ptr()


def _stream(stream=None) -> int:
    if stream is not None:
        return int(stream)
    import torch

    return torch.cuda.current_stream().cuda_stream


# ---- direct kernels (device tensors, asynchronous on the current stream) ----

def map_sin(x, y, stream=None):
    check(lib().mlkb_map_sin_f32(_ptr(x), _ptr(y), x.numel(), _stream(stream)))


def map_sin_dsin(x, y, dy, stream=None):
    check(lib().mlkb_map_sin_dsin_f32(_ptr(x), _ptr(y), _ptr(dy), x.numel(), _stream(stream)))


def map_chain(exprs: np.ndarray, a, out, b=None, scalars: Sequence[float] = (), poly7=False,
              stream=None):
    exprs = np.ascontiguousarray(exprs, dtype=kir.EXPR_DTYPE)
    sc = (C.c_double * max(1, len(scalars)))(*scalars)
    check(lib().mlkb_map_chain(exprs.ctypes.data, len(exprs), int(poly7), _ptr(a), _ptr(b),
                               _ptr(out), _dt_of(out), out.numel(), sc, len(scalars),
                               _stream(stream)))


def chain_compile(mode: int = -1):
    """Run-time chain compilation: mode 1 on, 0 off (interpreter), -1 query.
    Returns (active, compiled, launched): whether chains will be compiled and
    how many chain kernels this process has compiled and launched."""
    comp, launched = C.c_int64(0), C.c_int64(0)
    active = lib().mlkb_chain_compile(int(mode), C.byref(comp), C.byref(launched))
    return bool(active), comp.value, launched.value


def chain_build(exprs: np.ndarray, dtype: str = "f32", has_b: bool = False, poly7=False):
    """Compiles the kernel map_chain would use for this chain (no GPU needed)."""
    exprs = np.ascontiguousarray(exprs, dtype=kir.EXPR_DTYPE)
    check(lib().mlkb_chain_build(exprs.ctypes.data, len(exprs), int(poly7),
                                 F64 if dtype == "f64" else F32, int(has_b)))


def softmax(x, y, stream=None):
    rows, cols = x.shape
    fn = lib().mlkb_softmax_f32 if _dt_of(x) == F32 else lib().mlkb_softmax_f64
    check(fn(_ptr(x), _ptr(y), rows, cols, _stream(stream)))


def reducesum(x, y, stream=None):
    rows, cols = x.shape
    fn = lib().mlkb_reducesum_f32 if _dt_of(x) == F32 else lib().mlkb_reducesum_f64
    check(fn(_ptr(x), _ptr(y), rows, cols, _stream(stream)))


def gemm(a, b, c, accumulate=False, stream=None):
    m, k = a.shape
    k2, n = b.shape
    assert k == k2 and tuple(c.shape) == (m, n)
    dt = _dt_of(a)
    fn = {F16: lib().mlkb_gemm_f16_f32, F32: lib().mlkb_gemm_f32, F64: lib().mlkb_gemm_f64}[dt]
    check(fn(_ptr(a), _ptr(b), _ptr(c), m, n, k, int(accumulate), _stream(stream)))


def qk_softmax(q, k, y, scale: float, stream=None):
    batch, s, d = q.shape
    check(lib().mlkb_qk_softmax_f16(_ptr(q), _ptr(k), _ptr(y), batch, s, d, float(scale),
                                    _stream(stream)))


def qk_softmax_kt(q, kt, y, scale: float, stream=None):
    """Y[b] = softmax_rows(scale * Q[b] @ Kt[b]): Q [batch, m, d], Kt [batch, d, s]."""
    batch, m, d = q.shape
    s = kt.shape[2]
    assert tuple(kt.shape) == (batch, d, s) and tuple(y.shape) == (batch, m, s)
    check(lib().mlkb_qk_softmax_kt_f16(_ptr(q), _ptr(kt), _ptr(y), batch, m, s, d, float(scale),
                                       _stream(stream)))


# ---- attention (device tensors, 16-bit elements) ----------------------------------
# Unlike the entries above, these take strided views (only the last dimension
# contiguous) and run on their tensors' device, whichever device is current.

_HEADS = C.c_int64 * 24  # up to six mlkb_heads: data, rows, row stride, head stride
_HALF_DT = None


def _heads_args(tensors, names):
    """The operands as consecutive mlkb_heads, and their element type. Each is
    [rows, heads, d], or None."""
    global _HALF_DT
    if _HALF_DT is None:
        import torch

        _HALF_DT = {torch.float16: F16, torch.bfloat16: BF16}
    flat = []
    first = tensors[0]
    dtype, device = first.dtype, first.device
    if dtype not in _HALF_DT:
        raise ValueError(f"{names[0]}: dtype must be float16 or bfloat16, got {dtype}")
    for t, name in zip(tensors, names):
        if t is None:
            flat += (0, 0, 0, 0)
            continue
        if t.dtype is not dtype or t.device != device:
            raise ValueError(f"{name}: {t.dtype} on {t.device}, but {names[0]} is {dtype} on {device}")
        rows, heads, _ = t.shape
        row, head, last = t.stride()
        if last != 1 and t.shape[2] > 1:
            raise ValueError(f"{name}: the last dimension must be contiguous")
        flat += (t.data_ptr(), rows, row, head)
    return _HEADS(*flat), _HALF_DT[dtype]


def _int32_ptr(t, name, device, shape):
    import torch

    if t is None:
        return None
    if t.dtype is not torch.int32 or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous int32 on {device} needed")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {shape}")
    return t.data_ptr()


def _on_device(device, stream, call):
    """call(stream handle) with `device` current (the default stream is the
    device's current one)."""
    import torch

    if device.type != "cuda":
        raise ValueError(f"tensors must be on a CUDA device, not {device}")
    if device.index == torch.cuda.current_device():
        check(call(_stream(stream)))
    else:
        with torch.cuda.device(device):
            check(call(_stream(stream)))


def norm_rope(q, k, q_out, k_out, table, positions, sections=None, q_weight=None, k_weight=None,
              eps: float = 1e-6, interleaved: bool = False, stream=None):
    """Head norms (where weights are given) and position rotation of q
    [tokens, heads, d] and k [tokens, kv_heads, d] (k and k_out may be None)
    into q_out and k_out, which may be q and k themselves.

    table: f32 [positions, rot], cosines of the rot/2 angles, then sines.
    positions: int32 [tokens], or [axes, tokens] with `sections`, the number
    of pairs each axis turns. A token whose position is outside the table is
    left as it is (take_device_error() then reports it)."""
    import torch

    tokens, heads, d = q.shape
    kv = 0 if k is None else k.shape[1]
    ops, dt = _heads_args((q, k, q_out, k_out), ("q", "k", "q_out", "k_out"))
    device = q.device
    if q_out.shape != q.shape or (k is None) != (k_out is None) or (
            k is not None and (k_out.shape != k.shape or k.shape[0] != tokens or k.shape[2] != d)):
        raise ValueError("q_out and k_out must have the shapes of q and k, of equal tokens and d")
    if table.dtype is not torch.float32 or table.device != device or not table.is_contiguous() \
            or table.dim() != 2:
        raise ValueError("table: contiguous float32 [positions, rot] on the device of q needed")
    axes = 1 if positions.dim() == 1 else positions.shape[0]
    pos = _int32_ptr(positions, "positions", device,
                     (tokens,) if positions.dim() == 1 else (axes, tokens))
    if sections is not None and len(sections) != axes:
        raise ValueError(f"sections: {len(sections)} given for {axes} position axes")
    sec = (C.c_int32 * axes)(*sections) if sections is not None else None
    ptrs = []
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None and (w.dtype is not q.dtype or w.device != device or not w.is_contiguous()
                              or tuple(w.shape) != (d,)):
            raise ValueError(f"{name}: contiguous [{d}] of {q.dtype} on {device} needed")
        ptrs.append(None if w is None else w.data_ptr())
    table_rows, rot = table.shape
    _on_device(device, stream, lambda s: lib().mlkb_norm_rope(
        ops, C.byref(ops, 32), C.byref(ops, 64), C.byref(ops, 96), heads, kv, d, rot, ptrs[0], ptrs[1],
        eps, table.data_ptr(), table_rows, pos, tokens, sec, axes, int(interleaved), dt, s))


def attention_packed(q, k, v, y, q_starts, k_starts, scale: float, causal: bool = True, stream=None):
    """y = softmax(scale q k^T) v for each head, over packed sequences.

    q, y [rows, heads, d]; k, v [key rows, kv_heads, d]; q_starts, k_starts
    int32 [sequences + 1]: sequence s has the rows starts[s] .. starts[s+1]-1.
    causal: the last query of a sequence sees its last key. Rows of y outside
    the sequences are left as they were; a query that sees no key gets zeros."""
    ops, dt = _heads_args((q, k, v, y), ("q", "k", "v", "y"))
    rows, heads, d = q.shape
    kv = k.shape[1]
    if y.shape != q.shape or v.shape != k.shape or k.shape[2] != d:
        raise ValueError("y must have the shape of q, v that of k, and all the same d")
    device = q.device
    n = q_starts.shape[0]
    if n < 1:
        raise ValueError("q_starts: sequences + 1 entries needed")
    qs = _int32_ptr(q_starts, "q_starts", device, (n,))
    ks = _int32_ptr(k_starts, "k_starts", device, (n,))
    _on_device(device, stream, lambda s: lib().mlkb_attention_packed(
        ops, C.byref(ops, 32), C.byref(ops, 64), C.byref(ops, 96), heads, kv, d, qs, ks, n - 1,
        int(causal), scale, dt, s))


def attention_prefix_workspace(q, prefix_k, k_pages, pages=None) -> int:
    """Bytes of workspace attention_prefix needs for these operands."""
    import torch

    batch, steps, heads, d = q.shape
    wide = pages.shape[1] if pages is not None else min(1, k_pages.shape[0])
    with torch.cuda.device(q.device):
        return lib().mlkb_attention_prefix_workspace(batch, steps, heads, prefix_k.shape[1], d,
                                                     prefix_k.shape[0], k_pages.shape[1], wide)


def attention_prefix(q, prefix_k, prefix_v, k_pages, v_pages, y, lens, scale: float, pages=None,
                     workspace=None, stream=None):
    """Attention of a batch that shares a prefix: the newest tokens q [batch,
    steps, heads, d] of each request over the common keys prefix_k, prefix_v
    [prefix, kv_heads, d], then the request's own lens[b] keys, its newest
    tokens' among them and causal over those.

    k_pages, v_pages [pages, page size, kv_heads, d]; pages int32 [batch,
    pages a request may have] names them in order, or None: page b is request
    b's. lens int32 [batch]. workspace: a CUDA tensor of at least
    attention_prefix_workspace bytes, allocated here (on the current stream)
    when None."""
    import torch

    batch, steps, heads, d = q.shape
    kv = prefix_k.shape[1]
    page = k_pages.shape[1]
    if y.shape != q.shape or prefix_v.shape != prefix_k.shape or v_pages.shape != k_pages.shape \
            or prefix_k.shape[2] != d or tuple(k_pages.shape[2:]) != (kv, d):
        raise ValueError("y must have the shape of q, v that of k, and all the same d and kv heads")
    flat = [_flat2(t, n) for t, n in ((q, "q"), (k_pages, "k_pages"), (v_pages, "v_pages"), (y, "y"))]
    ops, dt = _heads_args((flat[0], prefix_k, prefix_v, flat[1], flat[2], flat[3]),
                          ("q", "prefix_k", "prefix_v", "k_pages", "v_pages", "y"))
    device = q.device
    wide = pages.shape[1] if pages is not None else min(1, k_pages.shape[0])
    if pages is None and k_pages.shape[0] not in (0, batch):
        raise ValueError("without a page table there must be one page for each request")
    table = _int32_ptr(pages, "pages", device, (batch, wide))
    own = _int32_ptr(lens, "lens", device, (batch,))

    def call(s):
        L = lib()
        ws = workspace
        if ws is None:
            need = L.mlkb_attention_prefix_workspace(batch, steps, heads, kv, d, prefix_k.shape[0],
                                                     page, wide)
            ws = torch.empty(max(need, 0), dtype=torch.uint8, device=device)
            if stream is not None:
                # the memory returns to the pool on the current stream: not before `stream` is done
                ws.record_stream(torch.cuda.ExternalStream(int(stream), device=device))
        elif ws.device != device or not ws.is_contiguous():
            raise ValueError(f"workspace: contiguous on {device} needed")
        return L.mlkb_attention_prefix(
            ops, C.byref(ops, 32), C.byref(ops, 64), C.byref(ops, 96), C.byref(ops, 128),
            C.byref(ops, 160), batch, steps, heads, kv, d, page, wide, table, own, scale, dt,
            ws.data_ptr(), ws.numel() * ws.element_size(), s)

    _on_device(device, stream, call)


def _flat2(t, name):
    """[a, b, heads, d] as [a * b, heads, d] without a copy."""
    a, b, heads, d = t.shape
    if a > 1 and b > 1 and t.stride(0) != b * t.stride(1):
        raise ValueError(f"{name}: its first two dimensions must have one common stride")
    row = t.stride(1) if b > 1 else t.stride(0)
    return t.as_strided((a * b, heads, d), (row, t.stride(2), t.stride(3)))


def fill(out, seed: int, stream_id: int, dist: str, lo: float, hi: float, stream=None):
    d = {"uniform": 0, "normal": 1}[dist]
    fn = lib().mlkb_fill_f32 if _dt_of(out) == F32 else lib().mlkb_fill_f16
    check(fn(_ptr(out), out.numel(), seed, stream_id, d, lo, hi, _stream(stream)))


def take_device_error() -> int:
    return lib().mlkb_take_device_error()


# ---- module API ---------------------------------------------------------------

class Module:
    """A Kernel IR module bound from its `mlk-kernel` JSON (dict or str)."""

    def __init__(self, module):
        text = module if isinstance(module, str) else kir.dumps(module)
        h = C.c_void_p()
        check(lib().mlkb_module_create(text.encode(), C.byref(h)))
        self._h = h

    def close(self) -> None:
        """Releases the native module (also done when the object is collected)."""
        if getattr(self, "_h", None):
            lib().mlkb_module_destroy(self._h)
            self._h = None

    def __del__(self):
        # At interpreter shutdown the module globals this needs may already be
        # gone; the process is exiting and the handle dies with it.
        try:
            self.close()
        except Exception:  # noqa: BLE001
            pass

    @property
    def kind(self) -> int:
        return lib().mlkb_module_kind(self._h)

    @property
    def num_buffers(self) -> int:
        return lib().mlkb_module_num_buffers(self._h)

    def plan(self, dtypes) -> str:
        """Names of the kernels run_dev launches with these buffer dtypes
        (MLKB_F16 / F32 / F64 codes, or arrays / tensors to take them from)."""
        codes = [d if isinstance(d, int) else _dt_of(d) for d in dtypes]
        arr = (C.c_int32 * len(codes))(*codes)
        buf = C.create_string_buffer(512)
        check(lib().mlkb_module_plan(self._h, arr, len(codes), buf, 512))
        return buf.value.decode()

    def _args(self, bufs, scalars):
        n = len(bufs)
        ptrs = (C.c_void_p * n)(*[_ptr(b) for b in bufs])
        dts = (C.c_int32 * n)(*[_dt_of(b) for b in bufs])
        sc = (C.c_double * max(1, len(scalars)))(*scalars)
        return ptrs, dts, n, sc

    def run_dev(self, bufs, n: int = 0, scalars: Sequence[float] = (), device=None,
                stream=None):
        """Runs over device tensors on `device` (default: the tensors' own
        device) and `stream` (default: torch's current stream of it)."""
        if device is None:
            device = next((b.device.index for b in bufs if hasattr(b, "device")), 0)
        if stream is None:
            import torch

            stream = torch.cuda.current_stream(device).cuda_stream
        ptrs, dts, nb, sc = self._args(bufs, scalars)
        check(lib().mlkb_module_run_dev(self._h, ptrs, dts, nb, n, sc, len(scalars), device,
                                        _stream(stream)))

    def run_host(self, bufs, n: int = 0, scalars: Sequence[float] = (), n_gpus: int = 0):
        ptrs, dts, nb, sc = self._args(bufs, scalars)
        check(lib().mlkb_module_run_host(self._h, ptrs, dts, nb, n, sc, len(scalars), n_gpus))

    def run_sharded(self, bufs, n: int = 0, scalars: Sequence[float] = (), n_gpus: int = 0,
                    assemble: bool = True, via_nccl: bool = False) -> int:
        """Inputs from host buffers, sharded over n_gpus devices; with
        `assemble` the outputs are device-0 tensors, filled by the shards'
        peer stores (maps) or by NCCL (other kinds, or with `via_nccl`).
        Returns the status (0 = ok) rather than raising, for fault-injection
        tests."""
        ptrs, dts, nb, sc = self._args(bufs, scalars)
        flags = (ASSEMBLE_DEVICE0 | (ASSEMBLE_VIA_NCCL if via_nccl else 0)) if assemble else 0
        return lib().mlkb_module_run_sharded(self._h, ptrs, dts, nb, n, sc, len(scalars), n_gpus,
                                             flags)


def legacy_call(module: dict, host_f64: Sequence[np.ndarray], n: int,
                scalars: Sequence[float] = ()) -> int:
    """Bind `module` and call mlk_kernel in the reference's legacy 1-D form
    (buffers..., n, scalars, n_scalars) exactly as LoadedKernel::run does;
    returns mlk_last_status()."""
    L = lib()
    check(L.mlk_bind_module(kir.dumps(module).encode()))
    sc = (C.c_double * max(1, len(scalars)))(*scalars)
    args = [b.ctypes.data for b in host_f64] + [n, C.cast(sc, C.c_void_p).value, len(scalars)]
    args += [0] * (18 - len(args))
    L.mlk_kernel(*args)
    return L.mlk_last_status()
