"""Python harness over the C ABI, with torch tensors as device buffers.

Mirrors the reference's entry points (source/q4rdna.cuh:5-24): each GEMV
call returns True when it launched and False when the call is not
applicable (the reference's ``return false``: nothing was launched and the
caller should use its own path).  Errors raise :class:`Q4RdnaError`.
Launches are asynchronous on torch's current stream of the tensors' device, or
on the stream whose handle is given as ``stream``; outputs that a call allocates
belong to the stream that it launches on.  All are forms for inference: none
has a backward.
"""
from __future__ import annotations

import ctypes
from typing import Iterable, Sequence

import torch

from . import _lib
from ._lib import (ALGO_SIDECAR, GLU_SWIGLU, GROUP, TILE_BYTES, TILE_ROWS, GemvDesc, LaunchOptions,
                   Q4RdnaError, Weight, check, load)


def packed_size(rows: int, cols: int) -> int:
    """Bytes of one packed tensor: rows*cols*34/64 (source/q4rdna.cu:149)."""
    return rows * cols * 34 // GROUP


# torch's current stream of a device index as a handle, without the Stream
# object that torch.cuda.current_stream builds around it: 0.08 us against
# 2.0 us, in a call whose kernel takes four.
try:
    _raw_stream = torch._C._cuda_getCurrentRawStream
except AttributeError:  # a torch build without this private function

    def _raw_stream(device: int) -> int:
        return torch.cuda.current_stream(device).cuda_stream


def _stream(device: torch.device | int | None = None) -> int:
    if isinstance(device, torch.device):
        device = device.index
    return _raw_stream(torch.cuda.current_device() if device is None else device)


def _on_stream(stream: int, device: int):
    """A context in which torch's current stream of the device is the one with
    this handle: a call that allocates its outputs does so there, since memory
    of another stream may still be in use by what is queued on that one."""
    if stream == 0:  # a handle of 0 would stand for a new stream
        return torch.cuda.stream(torch.cuda.default_stream(device))
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device))


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _f32_vec(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype != torch.float32 or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 CUDA tensor")
    return t


def _on_device(t: torch.Tensor, name: str, device: int) -> None:
    """The weight's device is where the kernels read and write: a buffer on
    another device is refused here rather than passed by address."""
    if t.get_device() != device:
        raise ValueError(f"{name} lives on cuda:{t.device.index}, the weight on cuda:{device}")


def _f32_buf(t: torch.Tensor, name: str, numel: int, device: int) -> torch.Tensor:
    """A device buffer the kernels read or write numel floats of: checked
    here, since the library sees only its address and a short or misplaced
    buffer would be read or written past its end on the GPU."""
    _f32_vec(t, name)
    if t.numel() != numel:
        raise ValueError(f"{name} holds {t.numel()} floats, {numel} are needed")
    _on_device(t, name, device)
    return t


def _options(split_k: int, kernel: int):
    """The launch options' address; None, which means the same, for the policy."""
    if split_k == 0 and kernel == _lib.KERNEL_POLICY:
        return None
    opts = LaunchOptions()
    opts.split_k = split_k
    opts.kernel = kernel
    return ctypes.byref(opts)


class QWeight:
    """A packed Q4_RDNA tensor resident on a GPU.

    ``tiles`` keeps the device buffer alive (a uint8 tensor of
    rows*cols*34/64 bytes) unless the weight views a sidecar's buffer, which
    the sidecar owns.
    """

    def __init__(self, raw: Weight, tiles: torch.Tensor | None = None, owner=None):
        self.raw = raw
        self.tiles = tiles
        self._owner = owner

    @classmethod
    def from_tiles(cls, tiles: torch.Tensor, rows: int, cols: int) -> "QWeight":
        if tiles.dtype != torch.uint8 or not tiles.is_cuda or not tiles.is_contiguous():
            raise ValueError("tiles must be a contiguous uint8 CUDA tensor")
        if tiles.numel() != packed_size(rows, cols):
            raise ValueError(f"tiles hold {tiles.numel()} bytes, {rows}x{cols} needs {packed_size(rows, cols)}")
        raw = Weight()
        check(load().q4rdna_weight_from_device(tiles.data_ptr(), rows, cols, tiles.device.index, ctypes.byref(raw)))
        return cls(raw, tiles)

    @property
    def rows(self) -> int:
        return self.raw.rows

    @property
    def cols(self) -> int:
        return self.raw.columns

    @property
    def device(self) -> int:
        return self.raw.device

    @property
    def nbytes(self) -> int:
        return packed_size(self.rows, self.cols)


def mul_mat(w: QWeight, x: torch.Tensor, y: torch.Tensor | None = None, stream: int | None = None):
    """y = W x.  Returns y, or None when the call is not applicable."""
    x = _f32_vec(x, "x")
    if y is None:
        if stream is not None:
            with _on_stream(stream, x.get_device()):
                return mul_mat(w, x)
        y = torch.empty(w.rows, dtype=torch.float32, device=x.device)
    _f32_vec(y, "y")
    device = w.raw.device
    _on_device(x, "x", device)
    _on_device(y, "y", device)
    s = _raw_stream(device) if stream is None else stream
    ok = check(load().q4rdna_mul_mat(ctypes.byref(w.raw), x.data_ptr(), x.numel(), y.data_ptr(), y.numel(), s))
    return y if ok else None


def mul_mat_add(w: QWeight, x: torch.Tensor, add: torch.Tensor, y: torch.Tensor | None = None,
                stream: int | None = None):
    """y = W x + add.  Returns y, or None when not applicable."""
    x = _f32_vec(x, "x")
    add = _f32_vec(add, "add")
    if y is None:
        if stream is not None:
            with _on_stream(stream, x.get_device()):
                return mul_mat_add(w, x, add)
        y = torch.empty(w.rows, dtype=torch.float32, device=x.device)
    _f32_vec(y, "y")
    device = w.raw.device
    _on_device(x, "x", device)
    _on_device(add, "add", device)
    _on_device(y, "y", device)
    s = _raw_stream(device) if stream is None else stream
    ok = check(load().q4rdna_mul_mat_add(ctypes.byref(w.raw), x.data_ptr(), x.numel(), add.data_ptr(), add.numel(),
                                         y.data_ptr(), y.numel(), s))
    return y if ok else None


def mul_mat_glu(up: QWeight, gate: QWeight, x: torch.Tensor, y: torch.Tensor | None = None,
                glu_op: int = GLU_SWIGLU, stream: int | None = None):
    """y = (W_up x) * silu(W_gate x).  Returns y, or None when not applicable."""
    x = _f32_vec(x, "x")
    if y is None:
        if stream is not None:
            with _on_stream(stream, x.get_device()):
                return mul_mat_glu(up, gate, x, glu_op=glu_op)
        y = torch.empty(up.rows, dtype=torch.float32, device=x.device)
    _f32_vec(y, "y")
    device = up.raw.device
    _on_device(x, "x", device)
    _on_device(y, "y", device)
    s = _raw_stream(device) if stream is None else stream
    ok = check(load().q4rdna_mul_mat_glu(ctypes.byref(up.raw), ctypes.byref(gate.raw), x.data_ptr(), x.numel(),
                                         glu_op, y.data_ptr(), y.numel(), s))
    return y if ok else None


def mul_mat_ex(w: QWeight, x: torch.Tensor, y: torch.Tensor, gate: QWeight | None = None,
               add: torch.Tensor | None = None, split_k: int = 0, stream: int | None = None,
               kernel: int = _lib.KERNEL_POLICY) -> bool:
    """GEMV with explicit launch options: split_k (0 = the shape policy),
    kernel (KERNEL_VALU, or 0 = the policy, which is that kernel, or
    KERNEL_SEQUENTIAL: the reference's old mapping, split_k 0 or 1)."""
    _f32_buf(x, "x", w.cols, w.device)
    _f32_buf(y, "y", w.rows, w.device)
    if add is not None:
        _f32_buf(add, "add", w.rows, w.device)
    if gate is not None and (gate.rows, gate.cols) != (w.rows, w.cols):
        raise ValueError("gate and weight shapes differ")
    s = _raw_stream(x.get_device()) if stream is None else stream
    return check(load().q4rdna_mul_mat_ex(ctypes.byref(w.raw), ctypes.byref(gate.raw) if gate else None,
                                          x.data_ptr(), _ptr(add), y.data_ptr(), _options(split_k, kernel), s))


def mul_mat_batch(w: QWeight, x: torch.Tensor, y: torch.Tensor, gate: QWeight | None = None,
                  add: torch.Tensor | None = None, split_k: int = 0, stream: int | None = None,
                  kernel: int = _lib.KERNEL_POLICY) -> bool:
    """n activation vectors against one weight, one launch: x [n][cols], y and
    add [n][rows] (contiguous float32 on the weight's device)."""
    if x.dim() != 2 or not x.is_contiguous() or x.dtype != torch.float32:
        raise ValueError("x must be a contiguous float32 [n, cols] tensor")
    if y.dim() != 2 or not y.is_contiguous() or y.dtype != torch.float32 or y.shape[0] != x.shape[0]:
        raise ValueError("y must be a contiguous float32 [n, rows] tensor")
    if x.shape[1] != w.cols or y.shape[1] != w.rows:
        raise ValueError("x / y shapes do not match the weight")
    if add is not None and (add.shape != y.shape or not add.is_contiguous() or add.dtype != torch.float32):
        raise ValueError("add must match y")
    device = w.raw.device
    for t, name in ((x, "x"), (y, "y"), (add, "add")):
        if t is not None and (not t.is_cuda or t.get_device() != device):
            raise ValueError(f"{name} must live on the weight's device cuda:{device}")
    s = _raw_stream(x.get_device()) if stream is None else stream
    return check(load().q4rdna_mul_mat_batch(ctypes.byref(w.raw), ctypes.byref(gate.raw) if gate else None,
                                             x.data_ptr(), x.shape[0], _ptr(add), y.data_ptr(),
                                             _options(split_k, kernel), s))


def mul_mat_group(items: Sequence[tuple], x: torch.Tensor, stream: int | None = None,
                  kernel: int = _lib.KERNEL_POLICY, split_k: int = 0) -> bool:
    """GEMVs sharing one activation x in one launch.  items: (weight, y) or
    (weight, y, gate_weight_or_None, add_or_None); every weight has
    x.numel() columns.  split_k: 0 = the shape policy for the group's total
    rows.  Returns False when not applicable."""
    if not 1 <= len(items) <= _lib.MAX_GROUP:
        raise ValueError(f"a group holds 1..{_lib.MAX_GROUP} GEMVs")
    descs = (_lib.GroupDesc * len(items))()
    for i, it in enumerate(items):
        w, y = it[0], it[1]
        gate = it[2] if len(it) > 2 else None
        add = it[3] if len(it) > 3 else None
        _f32_buf(x, "x", w.cols, w.device)
        _f32_buf(y, f"item {i} y", w.rows, w.device)
        if add is not None:
            _f32_buf(add, f"item {i} add", w.rows, w.device)
        if gate is not None and (gate.rows, gate.cols, gate.device) != (w.rows, w.cols, w.device):
            raise ValueError(f"item {i}: gate and weight differ in shape or device")
        descs[i].weight = w.raw
        descs[i].gate_tiles = gate.raw.tiles if gate is not None else None
        descs[i].add = _ptr(add)
        descs[i].y = y.data_ptr()
    s = _raw_stream(x.get_device()) if stream is None else stream
    return check(load().q4rdna_mul_mat_group(descs, len(items), x.data_ptr(), x.numel(), _options(split_k, kernel), s))


def policy_split_k(rows: int, cols: int, device: int = 0) -> int:
    return load().q4rdna_policy_split_k(rows, cols, device)


def pack(w: torch.Tensor, algorithm: int = ALGO_SIDECAR, out: torch.Tensor | None = None,
         stream: int | None = None) -> torch.Tensor:
    """Quantize fp32 W [rows, cols] on the GPU into Q4_RDNA tiles (uint8)."""
    if w.dtype != torch.float32 or not w.is_cuda or not w.is_contiguous() or w.dim() != 2:
        raise ValueError("w must be a contiguous 2-D float32 CUDA tensor")
    rows, cols = w.shape
    if out is None:
        if stream is not None:
            with _on_stream(stream, w.get_device()):
                return pack(w, algorithm)
        out = torch.empty(packed_size(rows, cols), dtype=torch.uint8, device=w.device)
    # The library sees only out's address: a short, mistyped or misplaced
    # buffer would be written past its end on the GPU.
    if out.dtype != torch.uint8 or not out.is_cuda or not out.is_contiguous():
        raise ValueError("out must be a contiguous uint8 CUDA tensor")
    if out.numel() != packed_size(rows, cols):
        raise ValueError(f"out holds {out.numel()} bytes, {rows}x{cols} packs into {packed_size(rows, cols)}")
    if out.device != w.device:
        raise ValueError(f"out lives on {out.device}, w on {w.device}")
    s = _raw_stream(w.get_device()) if stream is None else stream
    check(load().q4rdna_pack(w.data_ptr(), rows, cols, algorithm, out.data_ptr(), s))
    return out


def dequantize(w: QWeight, out: torch.Tensor | None = None, stream: int | None = None) -> torch.Tensor:
    """fp32 [rows, cols] = scale * code (the exact product)."""
    if out is None:
        if stream is not None:
            with _on_stream(stream, w.device):
                return dequantize(w)
        out = torch.empty((w.rows, w.cols), dtype=torch.float32, device=torch.device("cuda", w.device))
    _f32_buf(out, "out", w.rows * w.cols, w.device)
    s = _raw_stream(out.get_device()) if stream is None else stream
    check(load().q4rdna_dequantize(ctypes.byref(w.raw), out.data_ptr(), s))
    return out


class Sidecar:
    """A sidecar file uploaded to one device (library-owned weights)."""

    def __init__(self, handle: int, device: int):
        self._h = ctypes.c_void_p(handle)
        self.device = device

    @classmethod
    def open(cls, path: str, device: int = 0) -> "Sidecar":
        h = ctypes.c_void_p()
        check(load().q4rdna_sidecar_open(path.encode(), device, ctypes.byref(h)))
        return cls(h.value, device)

    @classmethod
    def from_bytes(cls, image: bytes, device: int = 0) -> "Sidecar":
        h = ctypes.c_void_p()
        buf = ctypes.create_string_buffer(image, len(image))
        check(load().q4rdna_sidecar_open_memory(ctypes.cast(buf, ctypes.c_void_p), len(image), device, ctypes.byref(h)))
        return cls(h.value, device)

    def close(self) -> None:
        if self._h is not None and self._h.value:
            load().q4rdna_sidecar_close(self._h)
        self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __len__(self) -> int:
        return load().q4rdna_sidecar_count(self._h)

    def entries(self):
        L = load()
        out = []
        for i in range(len(self)):
            name = ctypes.create_string_buffer(64)
            r, c = ctypes.c_uint32(), ctypes.c_uint32()
            off, size = ctypes.c_uint64(), ctypes.c_uint64()
            check(L.q4rdna_sidecar_entry(self._h, i, name, ctypes.byref(r), ctypes.byref(c), ctypes.byref(off),
                                         ctypes.byref(size)))
            out.append((name.value.decode(), r.value, c.value, off.value, size.value))
        return out

    def find(self, name: str, ne0: int, ne1: int) -> QWeight | None:
        """Weight by ggml name with the ne0 = columns, ne1 = rows check."""
        raw = Weight()
        if not check(load().q4rdna_find(self._h, name.encode(), ne0, ne1, ctypes.byref(raw))):
            return None
        return QWeight(raw, owner=self)

    def hits(self, index: int) -> int:
        """GEMV launches that streamed entry `index` (q4rdna_sidecar_hits)."""
        return int(load().q4rdna_sidecar_hits(self._h, index))


def launch_count() -> int:
    """GEMV kernel launches made through the library (q4rdna_launch_count)."""
    return int(load().q4rdna_launch_count())


def report_stats() -> None:
    """The reference's launch report on stderr (q4rdna_report_stats)."""
    load().q4rdna_report_stats()


def inspect_sidecar(image: bytes, file_size: int | None = None) -> int:
    """Validate a sidecar header + index on the host; returns the entry count."""
    count = ctypes.c_uint32()
    buf = ctypes.create_string_buffer(bytes(image), len(image))
    check(load().q4rdna_sidecar_inspect(ctypes.cast(buf, ctypes.c_void_p), len(image),
                                        len(image) if file_size is None else file_size, ctypes.byref(count)))
    return count.value


def scope_allows(scope: str | None, name: str) -> bool:
    return bool(load().q4rdna_scope_allows(None if scope is None else scope.encode(), name.encode()))


class Plan:
    """A multi-tensor GEMV sweep launched as one kernel."""

    def __init__(self, items: Sequence[tuple], device: int = 0, batch: int = 1):
        """items: (weight, x, y) or (weight, x, y, gate_weight_or_None, add_or_None).

        batch > 1: each x holds `batch` activation vectors ([batch, cols],
        contiguous), y and add hold [batch, rows]."""
        descs = (GemvDesc * len(items))()
        self._keep = []
        for i, it in enumerate(items):
            w, x, y = it[0], it[1], it[2]
            gate = it[3] if len(it) > 3 else None
            add = it[4] if len(it) > 4 else None
            if w.device != device:
                raise ValueError(f"item {i}: the weight lives on cuda:{w.device}, the plan on cuda:{device}")
            _f32_buf(x, f"item {i} x", batch * w.cols, device)
            _f32_buf(y, f"item {i} y", batch * w.rows, device)
            if add is not None:
                _f32_buf(add, f"item {i} add", batch * w.rows, device)
            if gate is not None and (gate.rows, gate.cols, gate.device) != (w.rows, w.cols, w.device):
                raise ValueError(f"item {i}: gate and weight differ in shape or device")
            descs[i].weight = w.raw
            descs[i].gate_tiles = gate.raw.tiles if gate is not None else None
            descs[i].x = x.data_ptr()
            descs[i].add = _ptr(add)
            descs[i].y = y.data_ptr()
            self._keep.append(it)
        h = ctypes.c_void_p()
        check(load().q4rdna_plan_create_batch(descs, len(items), batch, device, ctypes.byref(h)))
        self._h = h
        self.device = device
        self.batch = batch

    @property
    def workgroups(self) -> int:
        return load().q4rdna_plan_workgroups(self._h)

    def launch(self, stream: int | None = None) -> bool:
        """prepare() + sweep() on one stream."""
        s = _raw_stream(self.device) if stream is None else stream
        return check(load().q4rdna_plan_launch(self._h, s))

    def prepare(self, stream: int | None = None) -> bool:
        """Convert every activation into the plan's int8 digit buffers."""
        s = _raw_stream(self.device) if stream is None else stream
        return check(load().q4rdna_plan_prepare(self._h, s))

    def sweep(self, stream: int | None = None) -> bool:
        """Run the GEMVs (after a prepare of the same activations)."""
        s = _raw_stream(self.device) if stream is None else stream
        return check(load().q4rdna_plan_sweep(self._h, s))

    def close(self) -> None:
        if self._h is not None and self._h.value:
            load().q4rdna_plan_destroy(self._h)
        self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _dtype(t: torch.dtype) -> int:
    code = _DTYPES.get(t)
    if code is None:
        raise ValueError(f"dtype {t}: float32, float16 and bfloat16 are supported")
    return code


def _no_gradient(name: str) -> None:
    """For a tensor that requires a gradient: the calls have no backward, and
    their results would silently be constants to torch."""
    if torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which this call cannot give: use torch.no_grad() or detach it")


def _plain(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device: int) -> int:
    """The address of a contiguous tensor that the kernels read or write whole."""
    if t.requires_grad:
        _no_gradient(name)
    if t.dtype != dtype or t.get_device() != device or not t.is_contiguous() or t.shape != shape:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, shape: tuple, device: int) -> tuple[int, int, int]:
    """(address, token stride, head stride) of activations [tokens, heads, dim]."""
    if t.requires_grad:
        _no_gradient(name)
    if t.dtype != dtype or t.get_device() != device or t.shape != shape:
        raise ValueError(f"{name} must be a {dtype} tensor of shape {tuple(shape)} on cuda:{device}, got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    token_stride, head_stride, stride = t.stride()
    if stride != 1:
        raise ValueError(f"the numbers of a head of {name} must be contiguous")
    return t.data_ptr(), token_stride, head_stride


_NO_ROWS = (0, 0, 0)


def _packed_like(t: torch.Tensor) -> torch.Tensor:
    """What the calls allocate for an output where torch.empty_like, which lays
    a tensor out in the order of t's strides, would put the numbers of a row
    apart: t's rows overlap, as a sliding window's do."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _no_overlap(t: torch.Tensor, name: str) -> None:
    """An output whose rows share memory would be written by several rows at once."""
    if not t.is_contiguous():
        dims = sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1)
        reach = 1
        for st, n in dims:
            if st < reach:
                raise ValueError(f"rows of {name} overlap")
            reach = st * (n - 1) + reach


class KVBatch:
    """The sequences of one step (q4rdna_kv_batch), shared by all layers' calls.

    past [sequences], table [sequences, width] and, where given, cu_tokens
    [sequences + 1] and slots [sequences] are int32 CUDA tensors, read when
    the kernels run: a captured graph may be replayed after they were filled
    anew.  Without cu_tokens every sequence has one token; with it max_tokens
    (an int) bounds the tokens of a sequence, None where it is not known: a
    bound lets short steps take faster paths.

    The kernels refuse a sequence whose entries are out of range, and pages
    outside the cache, and count them in :meth:`KVCache.faults`.  A refused
    sequence's rows of an output are not written, nor are rows behind
    cu_tokens[-1]: in an output that a call allocated they hold whatever was in
    that memory.
    """

    def __init__(self, past: torch.Tensor, table: torch.Tensor, cu_tokens: torch.Tensor | None = None,
                 slots: torch.Tensor | None = None, max_tokens: int | None = None):
        if not past.is_cuda or past.dim() != 1 or table.dim() != 2:
            raise ValueError("past must be a CUDA tensor [sequences], table [sequences, width]")
        device, n = past.get_device(), past.shape[0]
        raw = _lib.BatchDesc()
        raw.past = _plain(past, "past", torch.int32, (n,), device)
        raw.table = _plain(table, "table", torch.int32, (n, table.shape[1]), device)
        if cu_tokens is not None:
            raw.cu_tokens = _plain(cu_tokens, "cu_tokens", torch.int32, (n + 1,), device)
            if max_tokens is None:
                max_tokens = 0xffffffff  # the calls' tokens bound them
        elif max_tokens is None:
            max_tokens = 1
        elif max_tokens != 1:
            raise ValueError("without cu_tokens every sequence has one token")
        if slots is not None:
            raw.slots = _plain(slots, "slots", torch.int32, (n,), device)
        if not 1 <= max_tokens < 1 << 32:
            raise ValueError("max_tokens must be at least 1 (and below 2^32)")
        raw.sequences = n
        raw.max_tokens = max_tokens
        raw.table_width = table.shape[1]
        self.raw = raw
        self._call = -1, None  # the last call's tokens and descriptor
        self.device = device
        self.sequences = n
        self._keep = (past, table, cu_tokens, slots)

    def _of(self, tokens: int):
        """The descriptor for a call on `tokens` tokens: a new one where the last
        call had another count (that call may still be using its own)."""
        held, step = self._call
        if held != tokens:
            if self._keep[2] is None and tokens != self.sequences:
                raise ValueError(f"{tokens} tokens for {self.sequences} sequences: without cu_tokens each has one")
            raw = _lib.BatchDesc.from_buffer_copy(self.raw)
            raw.tokens = tokens
            step = ctypes.byref(raw)
            self._call = tokens, step
        return step


class KVCache:
    """A layer's paged key/value cache in 8 bits (q4rdna_kv_cache).

    pages int8 [pages, kv_heads, 2, 64 * head_dim], scales float32 [pages,
    kv_heads, 2], open int8 [slots, 2, kv_heads, 4, 64 * head_dim] and
    open_scales float32 [slots, 2, kv_heads, 2, 64]; :meth:`empty` makes them.
    The format, and what a page and a slot hold, is described in
    include/q4rdna.h.
    """

    def __init__(self, pages: torch.Tensor, scales: torch.Tensor, open: torch.Tensor, open_scales: torch.Tensor):
        if pages.dim() != 4 or open.dim() != 5 or not pages.is_cuda:
            raise ValueError("pages must be a CUDA tensor [pages, kv_heads, 2, 64 * head_dim], open "
                             "[slots, 2, kv_heads, 4, 64 * head_dim]")
        device, (count, heads, _, size), slots = pages.get_device(), pages.shape, open.shape[0]
        if size % _lib.KV_BLOCK:
            raise ValueError("a block holds 64 * head_dim codes")
        raw = _lib.CacheDesc()
        raw.pages = _plain(pages, "pages", torch.int8, (count, heads, 2, size), device)
        raw.scales = _plain(scales, "scales", torch.float32, (count, heads, 2), device)
        raw.open = _plain(open, "open", torch.int8, (slots, 2, heads, 4, size), device)
        raw.open_scales = _plain(open_scales, "open_scales", torch.float32, (slots, 2, heads, 2, _lib.KV_BLOCK), device)
        self._faults = torch.zeros(1, dtype=torch.int32, device=pages.device)
        raw.faults = self._faults.data_ptr()
        raw.page_count, raw.slot_count, raw.kv_heads = count, slots, heads
        raw.head_dim = size // _lib.KV_BLOCK
        raw.device = device
        self.raw = raw
        self._ref = ctypes.byref(raw)
        self.device = device
        self.kv_heads = heads
        self.head_dim = raw.head_dim
        self.pages, self.scales, self.open, self.open_scales = pages, scales, open, open_scales

    @classmethod
    def empty(cls, pages: int, slots: int, kv_heads: int, head_dim: int, device: int = 0) -> "KVCache":
        dev = torch.device("cuda", device)
        size = _lib.KV_BLOCK * head_dim
        return cls(torch.zeros((pages, kv_heads, 2, size), dtype=torch.int8, device=dev),
                   torch.zeros((pages, kv_heads, 2), dtype=torch.float32, device=dev),
                   torch.zeros((slots, 2, kv_heads, 4, size), dtype=torch.int8, device=dev),
                   torch.zeros((slots, 2, kv_heads, 2, _lib.KV_BLOCK), dtype=torch.float32, device=dev))

    def faults(self) -> int:
        """How often the kernels refused a batch entry (waits for the device)."""
        return int(self._faults.item())

    def _step(self, batch: KVBatch, tokens: int):
        if batch.device != self.device:
            raise ValueError(f"the batch lives on cuda:{batch.device}, the cache on cuda:{self.device}")
        return batch._of(tokens)

    def append(self, batch: KVBatch, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
               interleaved: bool = False, q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
               eps: float = 1e-6, stream: int | None = None) -> torch.Tensor | None:
        """Append the step's k and v [tokens, kv_heads, head_dim]; returns q
        [tokens, q_heads, head_dim] normalised and rotated (q_norm, k_norm
        [head_dim]; cos, sin [positions, rotary / 2], float32).  Rows of a
        refused sequence are not written (see :class:`KVBatch`)."""
        if k.dim() != 3:
            raise ValueError("k must be [tokens, kv_heads, head_dim]")
        if stream is not None and q is not None and q_out is None:
            with _on_stream(stream, self.device):
                return self.append(batch, k, v, q, None, cos, sin, interleaved, q_norm, k_norm, eps)
        tokens, heads, dim, device, dtype = k.shape[0], self.kv_heads, self.head_dim, self.device, k.dtype
        step = self._step(batch, tokens)
        shape = (tokens, heads, dim)
        k_rows, v_rows = _rows(k, "k", dtype, shape, device), _rows(v, "v", dtype, shape, device)
        q_rows = out_rows = _NO_ROWS
        q_heads = 0
        if q is not None:
            if q.dim() != 3:
                raise ValueError("q must be [tokens, q_heads, head_dim]")
            q_heads = q.shape[1]
            shape = (tokens, q_heads, dim)
            q_rows = _rows(q, "q", dtype, shape, device)
            if q_out is None:
                q_out = torch.empty_like(q)
                token_stride, head_stride, stride = q_out.stride()
                if stride != 1:
                    q_out = _packed_like(q)
                    token_stride, head_stride, _ = q_out.stride()
                out_rows = q_out.data_ptr(), token_stride, head_stride
            else:
                _no_overlap(q_out, "q_out")
                out_rows = _rows(q_out, "q_out", dtype, shape, device)
        elif q_out is not None or q_norm is not None:
            raise ValueError("q_out or q_norm without q")
        cos_at = sin_at = positions = rotary = 0
        if cos is not None:
            table = cos.shape
            if len(table) != 2 or sin is None:
                raise ValueError("cos and sin must be [positions, rotary / 2]")
            cos_at = _plain(cos, "cos", torch.float32, table, device)
            sin_at = _plain(sin, "sin", torch.float32, table, device)
            positions, rotary = table[0], 2 * table[1]
        elif sin is not None:
            raise ValueError("sin without cos")
        q_weight = 0 if q_norm is None else _plain(q_norm, "q_norm", torch.float32, (dim,), device)
        k_weight = 0 if k_norm is None else _plain(k_norm, "k_norm", torch.float32, (dim,), device)
        d = _lib.APPEND.pack(_dtype(dtype), q_heads, *k_rows, *v_rows, *q_rows, *out_rows, cos_at, sin_at, positions,
                             rotary, interleaved, eps, q_weight, k_weight)
        s = _raw_stream(device) if stream is None else stream
        check(load().q4rdna_kv_append(self._ref, step, d, s))
        return q_out

    def attend(self, batch: KVBatch, q: torch.Tensor, out: torch.Tensor | None = None, scale: float | None = None,
               window: int = 0, lse: bool | torch.Tensor = False, stream: int | None = None):
        """Attention of the step's q [tokens, q_heads, head_dim] over the cache,
        after :meth:`append` of the same batch.  scale None: head_dim ** -0.5.
        window > 0: the last `window` tokens only.  lse True (or a float32
        tensor [tokens, q_heads]): returns (out, lse).  Rows of a refused
        sequence are not written (see :class:`KVBatch`)."""
        if q.dim() != 3:
            raise ValueError("q must be [tokens, q_heads, head_dim]")
        if stream is not None and (out is None or lse is True):
            with _on_stream(stream, self.device):
                return self.attend(batch, q, out, scale, window, lse)
        shape, dtype, device = q.shape, q.dtype, self.device
        tokens, heads, _ = shape
        step = self._step(batch, tokens)
        shape = (tokens, heads, self.head_dim)
        rows = _rows(q, "q", dtype, shape, device)
        if out is None:
            out = torch.empty_like(q)
            token_stride, head_stride, stride = out.stride()
            if stride != 1:
                out = _packed_like(q)
                token_stride, head_stride, _ = out.stride()
            out_rows = out.data_ptr(), token_stride, head_stride
        else:
            _no_overlap(out, "out")
            out_rows = _rows(out, "out", dtype, shape, device)
        if lse is True:
            lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device)
        if not 0 <= window < 1 << 32:
            raise ValueError("window must not be negative (or reach 2^32)")
        d = _lib.ATTEND.pack(_dtype(dtype), heads, *rows, *out_rows,
                             0 if lse is False else _plain(lse, "lse", torch.float32, (tokens, heads), device),
                             self.head_dim ** -0.5 if scale is None else scale, window)
        s = _raw_stream(device) if stream is None else stream
        check(load().q4rdna_kv_attend(self._ref, step, d, s))
        return out if lse is False else (out, lse)

    def read(self, batch: KVBatch, tokens: int, dtype: torch.dtype = torch.float32, k: torch.Tensor | None = None,
             v: torch.Tensor | None = None, stream: int | None = None):
        """(k, v) [tokens, kv_heads, head_dim]: the batch's tokens (past[i] on,
        up to the sequence's length) as numbers.  Rows of a refused sequence
        are not written (see :class:`KVBatch`)."""
        shape, device = (tokens, self.kv_heads, self.head_dim), self.device
        if stream is not None and (k is None or v is None):
            with _on_stream(stream, device):
                return self.read(batch, tokens, dtype, k, v)
        step = self._step(batch, tokens)
        if k is None:
            k = self.scales.new_empty(shape, dtype=dtype)
        else:
            _no_overlap(k, "k")
        if v is None:
            v = torch.empty_like(k)
            if v.stride(2) != 1:
                v = _packed_like(k)
        else:
            _no_overlap(v, "v")
        rows = [_lib.ROWS.pack(*_rows(t, name, dtype, shape, device)) for t, name in ((k, "k"), (v, "v"))]
        s = _raw_stream(device) if stream is None else stream
        check(load().q4rdna_kv_read(self._ref, step, _dtype(dtype), rows[0], rows[1], s))
        return k, v


def add_norm(residual: torch.Tensor, y: torch.Tensor | None, weight: torch.Tensor | None, *,
             post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None, scale: float = 1.0,
             eps: float = 1e-6, h: torch.Tensor | None = None, n: torch.Tensor | None = None,
             stream: int | None = None):
    """(h, n): h = residual + scale * gate * post(y), n = rms(h) * weight.

    residual, y, h and n are [rows, width] (any row stride) of one dtype; gate
    is [width] or [rows, width]; weight and post_weight are float32 [width].
    y None: h is residual itself and is not written.  weight None: no n.
    post_weight None: y as it is.  h and n may be given (h may be residual or
    y, n may be y)."""
    if residual.dim() != 2 or not residual.is_cuda:
        raise ValueError("residual must be a CUDA tensor [rows, width]")
    device, shape, dtype = residual.get_device(), residual.shape, residual.dtype
    width = shape[1]
    if stream is not None and (y is not None and h is None or weight is not None and n is None):
        with _on_stream(stream, device):
            return add_norm(residual, y, weight, post_weight=post_weight, gate=gate, scale=scale, eps=eps, h=h, n=n)

    def matrix(t, name):
        if t.requires_grad:
            _no_gradient(name)
        stride = t.stride()
        if t.dtype != dtype or t.get_device() != device or t.shape != shape or stride[1] != 1 and width > 1:
            raise ValueError(f"{name} must be a {dtype} tensor {tuple(shape)} with contiguous rows on cuda:{device}")
        return t.data_ptr(), stride[0]

    r_at, r_stride = matrix(residual, "residual")
    y_at = y_stride = gate_at = gate_stride = h_at = h_stride = n_at = n_stride = post_at = weight_at = 0
    if y is not None:
        y_at, y_stride = matrix(y, "y")
        if h is None:
            h = torch.empty_like(residual)
            h_stride, stride = h.stride()
            if stride != 1:
                h = _packed_like(residual)
                h_stride = width
            h_at = h.data_ptr()
        else:
            _no_overlap(h, "h")
            h_at, h_stride = matrix(h, "h")
        if gate is not None:
            if gate.dim() == 1:
                gate_at = _plain(gate, "gate", dtype, (width,), device)
            else:
                gate_at, gate_stride = matrix(gate, "gate")
        if post_weight is not None:
            post_at = _plain(post_weight, "post_weight", torch.float32, (width,), device)
    elif gate is not None or post_weight is not None or h is not None:
        raise ValueError("gate, post_weight or h without y")
    if weight is not None:
        if n is None:
            n = torch.empty_like(residual)
            n_stride, stride = n.stride()
            if stride != 1:
                n = _packed_like(residual)
                n_stride = width
            n_at = n.data_ptr()
        else:
            _no_overlap(n, "n")
            n_at, n_stride = matrix(n, "n")
        weight_at = _plain(weight, "weight", torch.float32, (width,), device)
    elif n is not None:
        raise ValueError("n without a weight")
    if width == 0:
        return (residual if h is None else h), n
    d = _lib.ADD_NORM.pack(_dtype(dtype), shape[0], width, scale, eps, 0, r_at, y_at, gate_at, h_at, n_at, r_stride,
                           y_stride, gate_stride, h_stride, n_stride, post_at, weight_at)
    s = _raw_stream(device) if stream is None else stream
    if torch.cuda.current_device() == device:
        check(load().q4rdna_add_norm(d, s))
    else:
        with torch.cuda.device(device):
            check(load().q4rdna_add_norm(d, s))
    return (residual if h is None else h), n
