"""Typed wrappers over the libmlkb200 C ABI.

Device buffers are passed as torch CUDA tensors (torch provides device memory
and streams only); every computation happens in libmlkb200.so. Host buffers
are numpy arrays or CPU tensors.
"""
from __future__ import annotations

import ctypes as C
import struct
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
# A decoding step calls them for microseconds of work, so what they do on the
# host counts: torch's bindings are looked up once, operands go in one array.

class _Torch:
    """What the calls below use of torch, bound on first use."""

    def __init__(self):
        import torch

        self.dtypes = {torch.float16: F16, torch.bfloat16: BF16}
        self.int32, self.float32, self.uint8 = torch.int32, torch.float32, torch.uint8
        self.empty, self.device = torch.empty, torch.cuda.device
        self.external_stream, self.default_stream = torch.cuda.ExternalStream, torch.cuda.default_stream
        self.stream = torch.cuda.stream
        self.current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        # the device's index and the stream's handle without what is around them, where torch has that
        self.raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)


_torch = None
_pack_heads = struct.Struct("4q").pack  # mlkb_heads: data, rows, row and head stride
_NO_HEADS = _pack_heads(0, 0, 0, 0)


def _bind():
    global _torch
    if _torch is None:
        _torch = _Torch()
    return _torch


def _heads(tensors, names):
    """The operands ([rows, heads, d] each, [a, b, heads, d] taken as [a * b,
    heads, d], or None) as mlkb_heads and their shapes, then their element type
    and the index of their device."""
    first = tensors[0]
    dtype, index = first.dtype, first.get_device()
    code = _bind().dtypes.get(dtype)
    if code is None:
        raise ValueError(f"{names[0]}: dtype must be float16 or bfloat16, got {dtype}")
    if index < 0:
        raise ValueError(f"{names[0]}: must be on a CUDA device, not {first.device}")
    heads, shapes, pack = [], [], _pack_heads
    for t in tensors:
        if t is None:
            heads.append(_NO_HEADS)
            shapes.append(None)
            continue
        if t.dtype is not dtype or t.get_device() != index:
            raise ValueError(f"{names[len(heads)]}: {t.dtype} on {t.device}, but {names[0]} is {dtype} on "
                             f"{first.device}")
        shape, strides = t.shape, t.stride()
        rows, row = shape[0], strides[0]
        if len(shape) == 4:
            if shape[1] > 1:
                row = strides[1]
                if rows > 1 and strides[0] != shape[1] * row:
                    raise ValueError(f"{names[len(heads)]}: its first two dimensions must have one common "
                                     "stride")
            rows *= shape[1]
        elif len(shape) != 3:
            raise ValueError(f"{names[len(heads)]}: {len(shape)} dimensions, expected [rows, heads, d]")
        if strides[-1] != 1 and shape[-1] > 1:
            raise ValueError(f"{names[len(heads)]}: the last dimension must be contiguous")
        heads.append(pack(t.data_ptr(), rows, row, strides[-2]))
        shapes.append(shape)
    return heads, shapes, code, index


def _int32(t, name, index, shape):
    if t is None:
        return None
    if t.dtype is not _torch.int32 or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous int32 on CUDA device {index} needed")
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {shape}")
    return t.data_ptr()


def _call(fn, args, index, stream):
    """fn(*args, stream) with device `index` current, on its current stream by default."""
    if index != _torch.current_device():
        with _torch.device(index):
            return _call(fn, args, index, stream)
    status = fn(*args, _torch.raw_stream(index) if stream is None else int(stream))
    if status != 0:
        check(status)


def norm_rope(q, k, q_out, k_out, table, positions, sections=None, q_weight=None, k_weight=None,
              eps: float = 1e-6, interleaved: bool = False, stream=None):
    """Head norms (where weights are given) and position rotation of q
    [tokens, heads, d] and k [tokens, kv_heads, d] (k and k_out may be None)
    into q_out and k_out, which may be q and k themselves.

    table: f32 [positions, rot], cosines of the rot/2 angles, then sines.
    positions: int32 [tokens], or [axes, tokens] with `sections`, the number
    of pairs each axis turns. A token whose position is outside the table is
    left as it is (take_device_error() then reports it)."""
    ops, shapes, dt, index = _heads((q, k, q_out, k_out), ("q", "k", "q_out", "k_out"))
    shape, keys, shape_out, keys_out = shapes
    tokens, heads, d = shape
    kv = 0
    if shape_out != shape or (k is None) != (k_out is None):
        raise ValueError("q_out and k_out must have the shapes of q and k")
    if k is not None:
        kv = keys[1]
        if keys != (tokens, kv, d) or keys_out != keys:
            raise ValueError("k and k_out must have the tokens and d of q")
    if table.dtype is not _torch.float32 or table.get_device() != index or not table.is_contiguous() \
            or table.dim() != 2:
        raise ValueError("table: contiguous float32 [positions, rot] on the device of q needed")
    table_rows, rot = table.shape
    axes = 1 if positions.dim() == 1 else positions.shape[0]
    pos = _int32(positions, "positions", index, (tokens,) if positions.dim() == 1 else (axes, tokens))
    sec = None
    if sections is not None:
        if len(sections) != axes:
            raise ValueError(f"sections: {len(sections)} given for {axes} position axes")
        sec = (C.c_int32 * axes)(*sections)
    weights = []
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None and (w.dtype is not q.dtype or w.get_device() != index or not w.is_contiguous()
                              or w.shape != (d,)):
            raise ValueError(f"{name}: contiguous [{d}] of {q.dtype} on the device of q needed")
        weights.append(None if w is None else w.data_ptr())
    _call(lib().mlkb_norm_rope,
          (*ops, heads, kv, d, rot, *weights, eps, table.data_ptr(), table_rows, pos, tokens, sec, axes,
           int(interleaved), dt), index, stream)


def attention_packed(q, k, v, y, q_starts, k_starts, scale: float, causal: bool = True,
                     workspace=None, stream=None):
    """y = softmax(scale q k^T) v for each head, over packed sequences.

    q, y [rows, heads, d]; k, v [key rows, kv_heads, d]; q_starts, k_starts
    int32 [sequences + 1]: sequence s has the rows starts[s] .. starts[s+1]-1.
    causal: the last query of a sequence sees its last key. Rows of y outside
    the sequences are left as they were; a query that sees no key gets zeros.
    workspace: a CUDA tensor of at least attention_packed_workspace bytes (few
    queries over many keys need one), allocated here (on `stream`) when None."""
    ops, shapes, dt, index = _heads((q, k, v, y), ("q", "k", "v", "y"))
    rows, heads, d = shapes[0]
    keys, kv, d_keys = shapes[1]
    if shapes[3] != shapes[0] or shapes[2] != shapes[1] or d_keys != d:
        raise ValueError("y must have the shape of q, v that of k, and all the same d")
    n = q_starts.shape[0]
    if n < 1:
        raise ValueError("q_starts: sequences + 1 entries needed")
    qs = _int32(q_starts, "q_starts", index, (n,))
    ks = _int32(k_starts, "k_starts", index, (n,))
    L = lib()
    ws, size = _workspace(workspace, L.mlkb_attention_packed_workspace,
                          (rows, keys, n - 1, heads, kv, d), q, index, stream)
    _call(L.mlkb_attention_packed,
          (*ops, heads, kv, d, qs, ks, n - 1, int(causal), scale, dt,
           None if ws is None else ws.data_ptr(), size), index, stream)


def attention_packed_workspace(q, k, q_starts) -> int:
    """Bytes of workspace attention_packed uses for these operands (0: none)."""
    rows, heads, d = q.shape
    with _bind().device(q.device):
        return lib().mlkb_attention_packed_workspace(rows, k.shape[0], q_starts.shape[0] - 1, heads,
                                                     k.shape[1], d)


def _workspace(given, size_of, shape, q, index, stream):
    """The caller's workspace, or one of size_of(*shape) bytes; and its size."""
    if given is not None:
        if given.get_device() != index or not given.is_contiguous():
            raise ValueError(f"workspace: contiguous on CUDA device {index} needed")
        return given, given.numel() * given.element_size()
    if index != _torch.current_device():
        with _torch.device(index):
            return _workspace(given, size_of, shape, q, index, stream)
    need = size_of(*shape)
    if need <= 0:
        return None, 0
    if stream is None or int(stream) == _torch.raw_stream(index):
        return _torch.empty(need, dtype=_torch.uint8, device=q.device), need
    # from the stream's own pool: what the memory held before, and holds next, is in its order
    s = _torch.external_stream(int(stream), device=q.device) if int(stream) else \
        _torch.default_stream(q.device)
    with _torch.stream(s):
        return _torch.empty(need, dtype=_torch.uint8, device=q.device), need


def attention_prefix_workspace(q, prefix_k, k_pages, pages=None) -> int:
    """Bytes of workspace attention_prefix needs for these operands."""
    batch, steps, heads, d = q.shape
    wide = pages.shape[1] if pages is not None else min(1, k_pages.shape[0])
    with _bind().device(q.device):
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
    attention_prefix_workspace bytes, allocated here (on `stream`) when None."""
    ops, shapes, dt, index = _heads((q, prefix_k, prefix_v, k_pages, v_pages, y),
                                    ("q", "prefix_k", "prefix_v", "k_pages", "v_pages", "y"))
    batch, steps, heads, d = shapes[0]
    prefix, kv, d_keys = shapes[1]
    count, page, kv_pages, d_pages = shapes[3]
    if shapes[5] != shapes[0] or shapes[2] != shapes[1] or shapes[4] != shapes[3] or d_keys != d \
            or kv_pages != kv or d_pages != d:
        raise ValueError("y must have the shape of q, v that of k, and all the same d and kv heads")
    if pages is None:
        if count not in (0, batch):
            raise ValueError("without a page table there must be one page for each request")
        wide = min(1, count)
    else:
        wide = pages.shape[1]
    table = _int32(pages, "pages", index, (batch, wide))
    own = _int32(lens, "lens", index, (batch,))
    L = lib()
    ws, size = _workspace(workspace, L.mlkb_attention_prefix_workspace,
                          (batch, steps, heads, kv, d, prefix, page, wide), q, index, stream)
    _call(L.mlkb_attention_prefix,
          (*ops, batch, steps, heads, kv, d, page, wide, table, own, scale, dt,
           None if ws is None else ws.data_ptr(), size), index, stream)


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
