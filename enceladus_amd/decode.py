"""The operators of a decoding step over a paged key-value cache, as hand-written HIP kernels.

    q = decode.append_kv(k, v, k_cache, v_cache, block_table, seq_lens, q=q, cos=cos, sin=sin)
    o = decode.paged_attention(q, k_cache, v_cache, block_table, seq_lens)
    logits = decode.adjust_logits(logits, tokens=tokens, token_lens=lens, repetition=1.1)

A cache is two arrays `[pages, page size, key heads, head dimension]`, in any order in memory
(`x.permute(0, 2, 1, 3)` of one that keeps a page's heads together is as good): the elements of
a head are adjacent, and both caches have the same strides. `block_table[b, i]` is the page of
sequence b's tokens `i * page size` on, `seq_lens[b]` its length with the new tokens.

Arrays are torch-ROCm tensors, `enceladus.Tensor`s or NumPy arrays (which are copied to the GPU
and back), on one device; the work goes to its current stream and nothing waits for it. What the
device alone knows is checked there: a page outside the cache is neither read nor written, a
length beyond the block table counts as the whole of it, a negative one as none. Nothing is kept
from one call for the next but compiled kernels, so calls on several streams and captured graphs
do not meet; a call inside a capture needs one before it, which loads the kernel. There are no
gradients.
"""

from __future__ import annotations

import ctypes
import math
import operator
import struct
import sys
import threading

import numpy as np

from enceladus_amd.runtime import compile as C
from enceladus_amd.runtime import debug as _trace
from enceladus_amd.runtime import device as D
from enceladus_amd.runtime import hip
from enceladus_amd.runtime import tensor as T
from enceladus_amd.runtime import timing as _timing
from enceladus_amd.runtime.jit import _errbuf
from enceladus_amd.runtime.probe import check_mfma_layout

__all__ = ["append_kv", "paged_attention", "adjust_logits"]

_SOURCES = hip.INCLUDE_DIR.parent / "kernels"
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2, "fp8": 1, "i32": 4}
_Q = {"fp32": 0, "fp16": 1, "bf16": 2}
MAX_HEAD_DIM = 256
MAX_TOKENS = 1 << 30               # of a block table's row: positions are 32-bit


# -- kernels -----------------------------------------------------------------------------

_lock = threading.Lock()
_texts: dict[str, str] = {}
_functions: dict[tuple, ctypes.c_void_p] = {}
_modules: dict[tuple, ctypes.c_void_p] = {}


def _source(file: str, macros: tuple) -> str:
    text = _texts.get(file)
    if text is None:
        text = _texts[file] = (_SOURCES / file).read_text()
    return "".join(f"#define {k} {v}\n" for k, v in macros) + text


def _is_cached(file: str, macros: tuple) -> bool:
    return C.is_cached(_source(file, macros), file.removesuffix(".hip"))


def _code(file: str, macros: tuple) -> bytes:
    return C.compile_code(_source(file, macros), file.removesuffix(".hip"))


def _function(file: str, macros: tuple, name: str, device: int):
    """The kernel `name` of a compiled source on `device`, which is the current one."""
    f = _functions.get((file, macros, name, device))
    if f is not None:
        return f
    if file in ("paged_attention.hip", "tree_attention.hip"):
        check_mfma_layout()
    with _lock:
        mod = _modules.get((file, macros, device))
        if mod is None:
            code = _code(file, macros)
            mod = ctypes.c_void_p()
            hip.call("ek_module_load", ctypes.create_string_buffer(code, len(code)), len(code),
                     ctypes.byref(mod))
            _modules[file, macros, device] = mod
        f = ctypes.c_void_p()
        hip.call("ek_module_function", mod, name.encode(), ctypes.byref(f))
        _functions[file, macros, name, device] = f
    return f


class _Plan:
    """A call as its arrays' types, shapes and strides and its options decide it: the kernels,
    their grids and the bytes of their arguments but for the addresses. `arrays` (name, array
    or None) are in the order of the kernels' pointers, and `written` are the ones that they
    write; a workspace's address, if there is one, comes last."""

    def __init__(self, file: str, macros: tuple, launches: list, arrays: list, written: set,
                 workspace: int, tail: bytes, apart=()):
        self.file, self.macros, self.launches = file, macros, launches
        self.written, self.workspace, self.tail = written, workspace, tail
        self.device = _device_of(arrays)
        torch = _torch()
        self.on_gpu = all(a is None or (a.device >= 0) for _, a in arrays)
        self.where = torch.device("cuda", self.device) if self.device >= 0 else None
        count = len(arrays) + (workspace > 0)
        self.kernarg = struct.Struct(f"<{count}Q{len(tail)}s")
        self.packed = struct.Struct(
            f"<Q{8 + _ITEM.size * len(launches)}s{count}Q{len(tail)}s")
        self.items = None
        # (output, input, whether the input itself will do), by place and with their spans
        self.apart = [(i, j, same, arrays[i][1].span(), arrays[j][1].span(),
                       arrays[i][0], arrays[j][0])
                      for i, j, same in apart if arrays[i][1] and arrays[j][1]]

    def check_apart(self, objs: list) -> None:
        """Refuses an output that overlaps an input."""
        for i, j, same, n, m, name, other in self.apart:
            a, b = _Array(name, objs[i]), _Array(other, objs[j])
            p, q = a.address(), b.address()
            if p < q + m and q < p + n:
                _apart(name, a, other, b, same)

    def functions(self, device: int) -> list:
        return [_function(self.file, self.macros, name, device)
                for name, _, _ in self.launches]

    def run(self, objs: list) -> None:
        """Launches the kernels for `objs` (in the order of the plan's arrays)."""
        if not self.on_gpu:
            return self._run_general(objs)
        self.run_at([0 if x is None else x.data_ptr() for x in objs])

    def run_at(self, ptrs: list) -> None:
        """The same for arrays on a GPU by their addresses (0 where there is none)."""
        device = self.device
        if _cuda.here() != device:
            with _torch().cuda.device(device):
                return self.run_at(ptrs)
        if self.workspace:
            keep = _cuda.empty(self.workspace, dtype=_cuda.uint8, device=self.where)
            ptrs.append(keep.data_ptr())
        stream = _cuda.stream(device)
        if _timing.current() is not None or _trace._active is not None:
            return self._launch(device, stream, self.kernarg.pack(*ptrs, self.tail))
        if self.items is None:
            self.items = _LIST.pack(len(self.launches), self.kernarg.size) + b"".join(
                _ITEM.pack(f.value, *grid, 1, block)
                for f, (_, grid, block) in zip(self.functions(device), self.launches))
        packed = self.packed.pack(stream, self.items, *ptrs, self.tail)
        err = _errbuf()
        if _cuda.launch_list(packed, len(packed), err, 1024):
            raise hip.HipError(f"ek_launch_list: {err.value.decode(errors='replace')}")

    def _run_general(self, objs: list) -> None:
        """With arrays on the host or of the framework's own: copied as a kernel's are."""
        torch = _torch()
        device = 0
        if torch is not None and torch.cuda.is_available():
            device = torch.cuda.current_device()
            if 0 <= self.device != device:
                with torch.cuda.device(self.device):
                    return self._run_general(objs)
        at = [i for i, x in enumerate(objs) if x is not None]
        got, bindings = T.bind_arrays([objs[i] for i in at],
                                      {k for k, i in enumerate(at) if i in self.written})
        ptrs = [0] * len(objs)
        for i, p in zip(at, got):
            ptrs[i] = p
        if self.workspace:
            keep = T.empty((self.workspace,), "uint8")
            ptrs.append(keep.ptr)
        self._launch(device, D.current_stream(), self.kernarg.pack(*ptrs, self.tail))
        T.complete_bindings(bindings)
        if self.workspace:
            hip.call("ek_stream_sync", D.current_stream() or None)   # before it is freed

    def _launch(self, device: int, stream: int, kernarg: bytes) -> None:
        timer = _timing.current()
        for fn, (name, grid, block) in zip(self.functions(device), self.launches):
            grid = (*grid, 1)
            if timer is not None:
                timer.launch(stream, fn, grid, block, kernarg, len(kernarg))
                continue
            t0 = _trace.before_launch(stream) if _trace._active is not None else None
            hip.call("ek_launch", stream or None, fn, *grid, block, 1, 1, 0, kernarg,
                     len(kernarg))
            if t0 is not None:
                _trace.after_launch(t0, stream, name, grid, block, 0)


_LIST = struct.Struct("<II")
_ITEM = struct.Struct("<Q4I")


class _Cuda:
    """What a plan's warm run calls, looked up once torch's GPU side is in use."""

    def __getattr__(self, name):
        torch = _torch()
        self.here = torch.cuda.current_device
        self.stream = lambda device: torch.cuda.current_stream(device).cuda_stream
        if hasattr(torch._C, "_cuda_getCurrentRawStream"):
            self.stream = torch._C._cuda_getCurrentRawStream
        if hasattr(torch._C, "_cuda_getDevice") and torch.cuda.is_initialized():
            self.here = torch._C._cuda_getDevice
        self.empty, self.uint8 = torch.empty, torch.uint8
        self.empty_like, self.dense = torch.empty_like, torch.contiguous_format
        self.tensor = torch.Tensor
        self.launch_list = hip.load_library().ek_launch_list
        return self.__dict__[name]


_cuda = _Cuda()

# Plans of the calls seen, by all that decides them (no address, and nothing of the arrays'
# contents); started over when there are many.
_plans: dict[tuple, tuple] = {}
_MOST_PLANS = 4096


def _keep(key, plan) -> None:
    if key is not None and plan.on_gpu:
        if len(_plans) >= _MOST_PLANS:
            _plans.clear()
        _plans[key] = plan


def _of(x):
    """What a plan depends on of an array on a GPU."""
    return x.dtype, x.shape, x.stride(), x.get_device()


def _like(x):
    """A new dense array of x's kind, shape, type and device."""
    return _cuda.empty_like(x, memory_format=_cuda.dense) if x.__class__ is _cuda.tensor else \
        T.new_empty(x)


# -- arguments ---------------------------------------------------------------------------

_torch_kinds: dict = {}


def _torch():
    torch = sys.modules.get("torch")
    if torch is not None and not _torch_kinds:
        _torch_kinds.update({torch.float32: "fp32", torch.float16: "fp16",
                             torch.bfloat16: "bf16", torch.int32: "i32"})
        if hasattr(torch, "float8_e4m3fn"):
            _torch_kinds[torch.float8_e4m3fn] = "fp8"
    return torch


class _Array:
    """An array argument: its element kind, shape, strides in elements and device (-1: the
    host, or the framework's own)."""

    __slots__ = ("obj", "kind", "shape", "strides", "device", "size")

    def __init__(self, name: str, obj):
        torch = _torch()
        self.obj = obj
        if torch is not None and isinstance(obj, torch.Tensor):
            if obj.device.type not in ("cuda", "cpu") or obj.layout is not torch.strided:
                raise ValueError(f"`{name}` is not a dense tensor on a GPU or the host")
            self.kind = _torch_kinds.get(obj.dtype, str(obj.dtype))
            self.shape, self.strides = tuple(obj.shape), obj.stride()
            self.device = obj.device.index if obj.device.type == "cuda" else -1
            if self.device < 0 and self.kind == "fp8":
                raise ValueError(f"`{name}` holds float8 values on the host: move it to the GPU")
        elif T.is_array_like(obj):
            self.kind = T.elem_dtype(obj).name
            self.shape, self.strides = tuple(obj.shape), T.element_strides(obj)
            self.device = -1
            if any(s < 0 for s in self.strides):
                raise ValueError(f"`{name}` has negative strides")
        else:
            raise TypeError(f"`{name}` must be an array, got {type(obj).__name__}")
        self.size = _SIZE.get(self.kind, 0)

    def span(self, first: int = 0) -> int:
        """Bytes from the first element to the last one's end (of dimensions `first` on)."""
        if 0 in self.shape:
            return 0
        return self.size * (1 + sum((n - 1) * s for n, s in
                                    zip(self.shape[first:], self.strides[first:])))

    def address(self) -> int:
        if isinstance(self.obj, T.Tensor):
            return self.obj.ptr
        if isinstance(self.obj, np.ndarray):
            return self.obj.__array_interface__["data"][0]
        return self.obj.data_ptr()


def _need(ok: bool, text: str) -> None:
    if not ok:
        raise ValueError(text)


def _array(name: str, obj, kinds, ndim: int, shape=None, dense: bool = True) -> _Array:
    """`obj` as an array of one of `kinds` and of `ndim` dimensions (`shape`: its extents,
    None where any will do), with adjacent elements in the last one when `dense`."""
    a = _Array(name, obj)
    if a.kind not in kinds:
        raise TypeError(f"`{name}` must hold {' or '.join(kinds)}, got {a.kind}")
    _need(len(a.shape) == ndim, f"`{name}` must have {ndim} dimensions, got shape {a.shape}")
    if shape is not None:
        _need(all(w is None or w == n for w, n in zip(shape, a.shape)),
              f"`{name}` must have shape "
              f"({', '.join('any' if w is None else str(w) for w in shape)}), got {a.shape}")
    if dense and a.shape[-1] > 1:
        _need(a.strides[-1] == 1, f"the last dimension of `{name}` must be contiguous "
                                  f"(strides {tuple(a.strides)})")
    return a


def _written(name: str, a: _Array) -> None:
    """Refuses an array whose elements share memory, or that may not be written."""
    _need(all(s != 0 or n <= 1 for n, s in zip(a.shape, a.strides)),
          f"`{name}` is written: it can't be an expanded view (strides {tuple(a.strides)})")
    if isinstance(a.obj, np.ndarray):
        _need(a.obj.flags.writeable, f"`{name}` is a read-only NumPy array")


def _apart(name: str, out: _Array, other: str, a: _Array, same_ok: bool = True) -> None:
    """Refuses an output that overlaps an input, unless it is the input itself."""
    p, q = out.address(), a.address()
    if same_ok and p == q and out.shape == a.shape and tuple(out.strides) == tuple(a.strides) \
            and out.size == a.size:
        return
    if p + out.span() <= q or q + a.span() <= p:
        return
    # rows side by side in one wider array
    step = out.strides[0] * out.size
    if step > 0 and step == a.strides[0] * a.size:
        at = (p - q) % step
        if a.span(1) <= at and at + out.span(1) <= step:
            return
    raise ValueError(f"`{name}` overlaps `{other}`")


def _steps(a: _Array) -> list:
    """(stride, extent, bytes behind it: of the further dimensions and an element, less one) of
    a's dimensions in bytes, the widest stride first."""
    dims = sorted(((s * a.size, n) for n, s in zip(a.shape, a.strides) if n > 1), reverse=True)
    rest = a.size - 1 + sum((n - 1) * s for s, n in dims)
    found = []
    for s, n in dims:
        rest -= (n - 1) * s
        found.append((s, n, rest))
    return found


def _meet(steps: list, size: int, gap: int) -> bool:
    """Whether an array of such `_steps` shares bytes with its like `gap` bytes further on: a
    difference of two of its elements' places is within an element of that."""
    gaps = [gap]
    for s, n, rest in steps:
        gaps = [g - i * s for g in gaps
                for i in range(max(1 - n, -((rest - g) // s)), min(n - 1, (g + rest) // s) + 1)]
    return any(abs(g) < size for g in gaps)


def _device_of(arrays) -> int:
    """The GPU that the arrays are on: torch's, or -1 where none says one. Refuses two."""
    found = {a.device for _, a in arrays if a is not None and a.device >= 0}
    _need(len(found) < 2, "the arrays are on different GPUs: " + ", ".join(
        f"`{n}` on {a.device}" for n, a in arrays if a is not None and a.device >= 0))
    return found.pop() if found else -1


def _caches(k_cache, v_cache, heads, dim, kinds):
    kc = _array("k_cache", k_cache, kinds, 4, (None, None, heads, dim))
    vc = _array("v_cache", v_cache, (kc.kind,), 4, kc.shape)
    _need(tuple(kc.strides) == tuple(vc.strides), "`k_cache` and `v_cache` must have the same "
          f"strides, got {tuple(kc.strides)} and {tuple(vc.strides)}")
    _need(0 < kc.shape[1] <= MAX_TOKENS, "a page of `k_cache` must hold at least one token, and "
          f"at most {MAX_TOKENS}")
    _need(kc.shape[0] < 1 << 31, f"`k_cache` has {kc.shape[0]} pages: ids are 32-bit")
    return kc, vc


def _sequences(block_table, seq_lens, batch):
    bt = _array("block_table", block_table, ("i32",), 2, (batch, None))
    sl = _array("seq_lens", seq_lens, ("i32",), 1, (batch,), dense=False)
    return bt, sl


def _capacity(bt: _Array, kc: _Array) -> int:
    n = bt.shape[1] * kc.shape[1]
    _need(n <= MAX_TOKENS, f"`block_table` covers {n} tokens of a sequence: at most "
                           f"{MAX_TOKENS} are supported")
    return n


def _page_division(page: int) -> tuple[int, int]:
    """(multiplier, shift) with n // page == (n * multiplier >> 32) >> shift for n < 2^31 and
    page > 1: with 2^(b - 1) < page <= 2^b the multiplier, 2^(31 + b) / page rounded up, is off
    by less than one in 2^31."""
    bits = (page - 1).bit_length()
    return ((1 << (31 + bits)) // page + 1) & 0xFFFFFFFF, max(bits - 1, 0)


def _head_dim(dim: int, cache: str) -> None:
    _need(0 < dim <= MAX_HEAD_DIM and dim % (16 if cache == "fp8" else 8) == 0,
          f"the head dimension must be a multiple of {16 if cache == 'fp8' else 8} up to "
          f"{MAX_HEAD_DIM}, got {dim}")


# Scales beyond these have no product or reciprocal in 32 bits.
_SCALES = 2.0 ** -60, 2.0 ** 60


def _positive(name: str, x: float) -> None:
    _need(_SCALES[0] <= x <= _SCALES[1],
          f"`{name}` must be a positive number from 2^-60 to 2^60, got {x}")


def _f32(x: float) -> float:
    """x as far as 32 bits reach: infinite beyond."""
    return math.copysign(math.inf, x) if abs(x) > 3.4028234e38 else x


def _round32(x: float) -> float:
    return struct.unpack("<f", struct.pack("<f", x))[0]


# -- appending to the cache ----------------------------------------------------------------

_APPEND = struct.Struct("<16q11i4f4x")
_TURNS = struct.Struct("<i2q4Q")       # after its last number: see `_append_plan`
MAX_AXES = 4


# Bytes of rows, more than the L2s hold together, from which on they move past the caches: 21152
# tokens of 48 bf16 heads of 128 take 104 us with plain accesses and 93 with these (97 with the
# stores alone, 104 with the loads alone); 256 x 128000 bf16 logits 36 us, and 31 with such stores
# (36 with the loads too, which the product that made the logits has left in a cache).
_STREAM_ROWS = 32 << 20


# Rows that a lane takes one after the other. 265 MB of fp32 tokens of 72 rows of 192, one row at
# a time: 109 us with all 72, 61 with 8 or 4, 70 with 2; the tokens above 93 us with 6, 90 with 4;
# 41 MB of 80 rows of 64, many at a time: 11.7 with 4, 13.1 with 3.
_ROUNDS = 4


def _vector(size: int, rotary: int, dim: int, interleaved: bool) -> int:
    """Elements of an access: up to 16 bytes, dividing each part of a head."""
    v = 16 // size
    parts = (rotary, dim) if interleaved else (rotary // 2, dim - rotary)
    while any(p % v for p in parts):
        v //= 2
    return v


def append_kv(k, v, k_cache, v_cache, block_table, seq_lens, *, cu_tokens=None, q=None,
              q_out=None, cos=None, sin=None, interleaved: bool = False, k_scale: float = 1.0,
              v_scale: float = 1.0, positions=None, pair_axes=None):
    """Writes new keys and values into a paged cache, the keys rotated by their positions,
    and returns the queries rotated likewise.

    Sequence b's new tokens are the rows `cu_tokens[b]` to `cu_tokens[b + 1]` (without
    `cu_tokens`, row b alone); they are its last ones, so that the i-th of n is at position
    `seq_lens[b] - n + i`. Rows of no sequence (padding behind the last, or before the first),
    and rows whose position is negative, not covered by the block table or not in `cos`, or
    whose page is not in the cache, are skipped: neither cache nor `q_out` is written for them
    (a new `q_out` holds anything there). Two rows must not share a slot of the cache, and the
    new keys and values must not lie in it. The caches may lie in one array, as long as they
    share no element.

    With `cos` and `sin`, the first R elements of each key and query head are rotated in pairs,
    (j, j + R / 2), or (2 j, 2 j + 1) when `interleaved`: (x, y) becomes
    (x cos - y sin, y cos + x sin). They are those of the row's position, or, with `positions`, of
    positions of its own, wherever its slot is: one (the depth of a drafted token), or one on each
    of several axes (the time, height and width of a part of a picture or a video), of which pair
    j turns by the one on axis `pair_axes[j]`.

    Args:
        k, v: `[tokens, key heads, dim]`, float32, float16 or bfloat16; `dim` a multiple of 8
            up to 256 (of 16 with a float8 cache).
        k_cache, v_cache: `[pages, page size, key heads, dim]` of the type of `k`, or
            float8_e4m3fn; written in place.
        block_table: int32 `[batch, pages of a sequence]`.
        seq_lens: int32 `[batch]`, counting the new tokens.
        cu_tokens: int32 `[batch + 1]`, not descending.
        q: queries `[tokens, heads, dim]` of the type of `k`, to be rotated beside the keys.
        q_out: where the rotated queries go (`q` itself will do); new without it.
        cos, sin: float32 `[positions, R / 2]`.
        k_scale, v_scale: cached values are divided by these (float8: then saturated to +-448).
        positions: int32 `[tokens]`, or `[axes, tokens]` with at most 4 axes: rows of `cos` and
            `sin`. A row with a position that is not in them is skipped.
        pair_axes: R / 2 numbers, each pair's axis; needed with more than one. Where the axes of
            neighbouring pairs are equal in whole vectors (8 16-bit elements, 4 of 32), cos and
            sin are read in vectors too.

    Returns:
        The rotated queries, or None without `q`.
    """
    # plain numbers from here on: a plan is kept by their values
    interleaved, k_scale, v_scale = bool(interleaved), float(k_scale), float(v_scale)
    if pair_axes is not None:
        pair_axes = tuple(map(operator.index, pair_axes))
    try:
        key = (0, k.dtype, k.shape, k.stride(), k.get_device(), v.dtype, v.shape, v.stride(),
               v.get_device(), k_cache.dtype, k_cache.shape, k_cache.stride(),
               k_cache.get_device(), v_cache.dtype, v_cache.shape, v_cache.stride(),
               v_cache.get_device(), block_table.dtype, block_table.shape,
               block_table.stride(), block_table.get_device(), seq_lens.dtype, seq_lens.shape,
               seq_lens.stride(), seq_lens.get_device(),
               None if cu_tokens is None else _of(cu_tokens),
               None if q is None else (q.dtype, q.shape, q.stride(), q.get_device()),
               None if q_out is None else _of(q_out),
               None if cos is None else (cos.dtype, cos.shape, cos.stride(), cos.get_device()),
               None if sin is None else (sin.dtype, sin.shape, sin.stride(), sin.get_device()),
               interleaved, k_scale, v_scale)
        if positions is not None or pair_axes is not None:
            key += None if positions is None else _of(positions), pair_axes
        plan = _plans.get(key)
    except (AttributeError, TypeError, RuntimeError):
        key = plan = None              # arrays of another kind, or no arrays
    given = q_out is not None
    if plan is not None:
        gap = v_cache.data_ptr() - k_cache.data_ptr()
        if abs(gap) < plan.cache_span:
            if plan.cache_steps is None:
                plan.cache_steps = _steps(_Array("k_cache", k_cache))
            if _meet(plan.cache_steps, k_cache.element_size(), gap):
                plan = None            # refused below
    if plan is None:
        plan, q_out = _append_plan(k, v, k_cache, v_cache, block_table, seq_lens, cu_tokens, q,
                                   q_out, cos, sin, interleaved, k_scale, v_scale, positions,
                                   pair_axes)
        if plan is None:
            return q_out
        _keep(key, plan)
    elif q is not None and not given:
        q_out = _like(q)
    arrays = [q, k, v, q_out, k_cache, v_cache, block_table, seq_lens, cu_tokens, cos, sin]
    if positions is not None:
        arrays.append(positions)
    if given:
        plan.check_apart(arrays)
    plan.run(arrays)
    return q_out


def _turns(positions, pair_axes, tokens: int, pairs: int, vec: int):
    """(positions' array, macro, the numbers that the kernel has of them) for `pairs` rotated
    pairs, `vec` of them to a vector."""
    _need(positions is not None, "`pair_axes` is given without `positions`")
    _need(pairs > 0, "`positions` need `cos` and `sin`")
    a = _Array("positions", positions)
    one = len(a.shape) == 1
    a = _array("positions", positions, ("i32",), 1, (tokens,), dense=False) if one else \
        _array("positions", positions, ("i32",), 2, (None, tokens), dense=False)
    axes = 1 if one else a.shape[0]
    _need(0 < axes <= MAX_AXES, f"`positions` may have 1 to {MAX_AXES} axes, got {axes}")
    _need(pair_axes is not None or axes == 1, f"`positions` of {axes} axes need `pair_axes`")
    if pair_axes is None:
        pair_axes = (0,) * pairs
    _need(len(pair_axes) == pairs, f"`pair_axes` must have {pairs} entries, got {len(pair_axes)}")
    _need(all(0 <= x < axes for x in pair_axes), f"`pair_axes` must be from 0 to {axes - 1}")
    words = [sum(x << 2 * i for i, x in enumerate(pair_axes[w * 32:w * 32 + 32]))
             for w in range(4)]
    same = all(len(set(pair_axes[i:i + vec])) == 1 for i in range(0, pairs, vec))
    step = a.strides[0] if one else a.strides[1]
    return a, 1 if same else 2, (axes, 0 if one else a.strides[0], step, *words)


def _append_plan(k, v, k_cache, v_cache, block_table, seq_lens, cu_tokens, q, q_out, cos, sin,
                 interleaved, k_scale, v_scale, positions, pair_axes):
    """The checked call's plan (None: nothing to do) and its `q_out`."""
    ka = _array("k", k, ("fp32", "fp16", "bf16"), 3)
    tokens, kv_heads, dim = ka.shape
    _need(tokens <= 1 << 25, f"at most {1 << 25} tokens are supported, got {tokens}")
    va = _array("v", v, (ka.kind,), 3, ka.shape)
    kc, vc = _caches(k_cache, v_cache, kv_heads, dim, (ka.kind, "fp8"))
    _head_dim(dim, kc.kind)
    cu = None
    batch = tokens
    if cu_tokens is not None:
        cu = _array("cu_tokens", cu_tokens, ("i32",), 1, dense=False)
        _need(cu.shape[0] > 0, "`cu_tokens` must have one entry more than there are sequences")
        batch = cu.shape[0] - 1
    _need(batch <= 1 << 25, f"at most {1 << 25} sequences are supported, got {batch}")
    bt, sl = _sequences(block_table, seq_lens, batch)
    capacity = _capacity(bt, kc)
    qa = qo = None
    heads = 0
    if q is not None:
        qa = _array("q", q, (ka.kind,), 3, (tokens, None, dim))
        heads = qa.shape[1]
        if q_out is None:
            q_out = T.new_empty(q)
        qo = _array("q_out", q_out, (ka.kind,), 3, qa.shape)
        _written("q_out", qo)
    else:
        _need(q_out is None, "`q_out` is given without `q`")
    _written("k_cache", kc)
    _written("v_cache", vc)
    gap, steps = vc.address() - kc.address(), None
    if abs(gap) < kc.span():
        _need(gap != 0, "`k_cache` and `v_cache` are the same")
        steps = _steps(kc)
        _need(not _meet(steps, kc.size, gap), "`k_cache` overlaps `v_cache`")
    _need((cos is None) == (sin is None), "`cos` and `sin` go together")
    ca = sa = None
    rotary = 0
    if cos is not None:
        ca = _array("cos", cos, ("fp32",), 2)
        sa = _array("sin", sin, ("fp32",), 2, ca.shape)
        rotary = 2 * ca.shape[1]
        _need(0 < rotary <= dim, f"`cos` rotates {rotary} elements of heads of {dim}")
    _positive("k_scale", k_scale)
    _positive("v_scale", v_scale)
    arrays = [("q", qa), ("k", ka), ("v", va), ("q_out", qo), ("k_cache", kc), ("v_cache", vc),
              ("block_table", bt), ("seq_lens", sl), ("cu_tokens", cu), ("cos", ca),
              ("sin", sa)]
    interleaved = bool(interleaved) and rotary > 0
    vec = _vector(ka.size, rotary, dim, interleaved)
    turned = None
    if positions is not None or pair_axes is not None:
        turned = _turns(positions, pair_axes, tokens, rotary // 2,
                        max(1, vec // 2) if interleaved else vec)
        arrays.append(("positions", turned[0]))
    _device_of(arrays)
    if tokens == 0 or batch == 0 or kv_heads + heads == 0 or capacity == 0 or kc.shape[0] == 0:
        return None, q_out
    rows = heads + 2 * kv_heads
    macros = (("EK_Q", _Q[ka.kind]), ("EK_FP8", int(kc.kind == "fp8")), ("EK_V", vec),
              ("EK_PAIRS", int(interleaved)),
              ("EK_STREAM", int(tokens * rows * dim * ka.size > _STREAM_ROWS)))
    if turned:
        macros += (("EK_AXES", turned[1]),)
    # Waves per token: as many as it has rows for while CUs are without one, then enough for
    # _ROUNDS rows a lane (2^25 in all: a grid holds fewer than 2^32 threads).
    places = dim // vec if interleaved else (dim - rotary // 2) // vec
    most = -(-rows // max(1, 64 // places))
    parts = max(1, min(most, 4096 // tokens), min(-(-most // _ROUNDS), (1 << 25) // tokens))
    zero = (0, 0, 0)
    qs, os = (a.strides if a is not None else zero for a in (qa, qo))
    tail = _APPEND.pack(
        qs[0], qs[1], ka.strides[0], ka.strides[1], va.strides[0], va.strides[1], os[0], os[1],
        *(s * kc.size for s in kc.strides[:3]), bt.strides[0], sl.strides[0],
        cu.strides[0] if cu else 0, ca.strides[0] if ca else 0, sa.strides[0] if sa else 0,
        tokens, batch, heads, kv_heads, dim, rotary, kc.shape[1], kc.shape[0], capacity,
        ca.shape[0] if ca else 0, parts, k_scale, v_scale, 1.0 / _round32(k_scale),
        1.0 / _round32(v_scale))
    if turned:
        tail = tail[:-4] + _TURNS.pack(*turned[2])
    plan = _Plan("append_kv.hip", macros,
                 [("ek_append_kv", (-(-tokens * parts // 4), 1), 256)], arrays, {3, 4, 5}, 0,
                 tail, [(3, 0, True), (3, 1, False), (3, 2, False), (3, 4, False),
                        (3, 5, False)] + ([(3, 11, False)] if turned else []))
    plan.cache_span, plan.cache_steps = kc.span(), steps
    return plan, q_out


# -- attention over the cache ----------------------------------------------------------------

_ATTEND = struct.Struct("<9q8iI4iI3f4x")
_UNIT = 16                          # tokens: what a sequence is split in multiples of
_MIN_UNITS = 4                      # of a chunk
_STREAM = 256 << 20                # bytes of caches that do not stay in the last-level cache
# Chunks of all sequences and key heads, per CU: two waves per SIMD. More of them leave more
# partial results (one sequence of 131075, fp16: 94.8 us with 8, 102.3 with 16), fewer leave loads
# out (100.4 with 6), and any that do not fit the SIMDs evenly run longer (64 ragged sequences,
# bf16: 88.3 with 8, 96.2 with 10).
_WAVES = 8


def _step(width: int, size: int, short: bool) -> int:
    """Keys per wave and step: 8 KB of keys and values, where there are 16 to 32 keys in that; of
    an e4m3 cache twice as many, whose conversions and scores cost more per byte than their loads.
    Measured at their best numbers of waves: 64 ragged sequences, 501 MB of bf16, heads of 128:
    16 keys 87.7 us, 32 89.8 (and 187 registers instead of 128), 64 118; 24 ragged sequences, 153 MB
    of e4m3: 16 keys 50.7 us, 32 46.4, 64 43.4. `short`: no wave will have many, so that fewer waits
    count for more: one sequence of 1999 tokens, bf16 10.7 us with 16 keys, 9.9 with 32, 11.1 with 64;
    46 sequences of at most 317 12.4, 11.4 and 14.1."""
    if size == 1:
        return max(16, min(64, 8192 // width))
    if short and width * size == 256:
        return 32
    return max(16, min(32, 4096 // (width * size)))


def paged_attention(q, k_cache, v_cache, block_table, seq_lens, *, scale: float | None = None,
                    window: int = 0, softcap: float = 0.0, k_scale: float = 1.0,
                    v_scale: float = 1.0, out=None, return_lse: bool = False):
    """Attention of one token per sequence over a paged cache (which holds its own key and
    value already).

    For query head h of sequence b: s_j = `scale` * q . k_j over the sequence's tokens, of
    which only the last `window` count when that is above 0, made `softcap` * tanh(s_j /
    `softcap`) when that is above 0; the result is the sum of softmax(s)_j v_j. `heads` is a
    multiple of the key heads: head h reads key head h // (heads / key heads). A sequence
    without tokens, or with no score above -inf, gives zeros. Tokens on a page outside the cache count as absent. Cache
    memory that no sequence's length reaches may hold anything, NaN included. A value among a
    sequence's own that is not finite makes its element of the result infinite or NaN.

    Args:
        q: `[batch, heads, dim]`, float32, float16 or bfloat16; `dim` a multiple of 8 up to
            256 (of 16 with a float8 cache); at most 65536 sequences (every wave looks for its
            own among them, which is most of the time from some thousand short ones on).
        k_cache, v_cache: `[pages, page size, key heads, dim]` of the type of `q`, or
            float8_e4m3fn (not with float32).
        block_table: int32 `[batch, pages of a sequence]`.
        seq_lens: int32 `[batch]`.
        scale: of the scores; 1 / sqrt(dim) without it.
        k_scale, v_scale: what cached values are multiplied by.
        out: where the result goes (`q` itself will do); new without it.
        return_lse: also return the log of each head's sum of exp(s_j), float32
            `[batch, heads]` (-inf without tokens), by which results over parts of a sequence
            are joined.

    Returns:
        The result, `[batch, heads, dim]` of the type of `q`; `(result, lse)` when
        `return_lse`.
    """
    # plain numbers from here on: a plan is kept by their values
    scale = None if scale is None else float(scale)
    window, softcap = operator.index(window), float(softcap)
    k_scale, v_scale = float(k_scale), float(v_scale)
    try:
        key = (1, q.dtype, q.shape, q.stride(), q.get_device(), k_cache.dtype, k_cache.shape,
               k_cache.stride(), k_cache.get_device(), v_cache.dtype, v_cache.shape,
               v_cache.stride(), v_cache.get_device(), block_table.dtype, block_table.shape,
               block_table.stride(), block_table.get_device(), seq_lens.dtype, seq_lens.shape,
               seq_lens.stride(), seq_lens.get_device(), None if out is None else _of(out),
               scale, window, softcap, k_scale, v_scale)
        plan = _plans.get(key)
    except (AttributeError, TypeError, RuntimeError):
        key = plan = None              # arrays of another kind, or no arrays
    given = out is not None
    if plan is None:
        plan, out = _attention_plan(q, k_cache, v_cache, block_table, seq_lens, scale, window,
                                    softcap, k_scale, v_scale, out)
        if plan is not None:
            _keep(key, plan)
    elif not given:
        out = _like(q)
    lse = T.new_empty(q, tuple(q.shape[:2]), np.float32) if return_lse else None
    if plan is not None:
        arrays = [q, k_cache, v_cache, block_table, seq_lens, out, lse]
        if given:
            plan.check_apart(arrays)
        plan.run(arrays)
    return (out, lse) if return_lse else out


def _attention_plan(q, k_cache, v_cache, block_table, seq_lens, scale, window, softcap, k_scale,
                    v_scale, out):
    """The checked call's plan (None: nothing to do) and its `out`."""
    qa = _array("q", q, ("fp32", "fp16", "bf16"), 3)
    batch, heads, dim = qa.shape
    kc, vc = _caches(k_cache, v_cache, None, dim,
                     (qa.kind,) if qa.kind == "fp32" else (qa.kind, "fp8"))
    kv_heads = kc.shape[2]
    _head_dim(dim, kc.kind)
    _need(kv_heads > 0 and heads % kv_heads == 0,
          f"{heads} query heads are not a multiple of {kv_heads} key heads")
    _need(heads <= 65535 and batch <= 1 << 16,
          f"at most 65535 query heads and {1 << 16} sequences are supported, got {heads}, {batch}")
    bt, sl = _sequences(block_table, seq_lens, batch)
    capacity = _capacity(bt, kc)
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    _need(abs(scale) <= _SCALES[1], f"`scale` must be at most 2^60, got {scale}")
    _need(softcap == 0 or _SCALES[0] <= softcap <= _SCALES[1],
          f"`softcap` must be 0 or from 2^-60 to 2^60, got {softcap}")
    _need(window >= 0, f"`window` must be at least 0, got {window}")
    _positive("k_scale", k_scale)
    _positive("v_scale", v_scale)
    if out is None:
        out = T.new_empty(q)
    oa = _array("out", out, (qa.kind,), 3, qa.shape)
    _written("out", oa)
    arrays = [("q", qa), ("k_cache", kc), ("v_cache", vc), ("block_table", bt),
              ("seq_lens", sl), ("out", oa), ("lse", None)]
    _device_of(arrays)
    if batch == 0 or heads == 0:
        return None, out
    if kc.shape[0] == 0:
        capacity = 0
    window = min(window, MAX_TOKENS)
    most = -(-(min(window, capacity) if window else capacity) // _UNIT)
    _need(batch * most < 1 << 31, f"`block_table` covers {batch} sequences of {capacity} tokens: "
          f"at most {_UNIT << 31} tokens in all are supported")
    group = heads // kv_heads
    y = kv_heads * (-(-group // 16))
    items = max(1, min(_WAVES * C.coarsen_cap() // y, batch * -(-most // _MIN_UNITS)))
    width = 64 if dim <= 64 else 128 if dim <= 128 else 256
    macros = (("EK_Q", _Q[qa.kind]), ("EK_FP8", int(kc.kind == "fp8")), ("EK_DP", width),
              ("EK_PAD", int(dim != width)),
              ("EK_KT", _step(width, kc.size, batch * most <= 8 * items)))
    log2e = 1.4426950408889634
    # Heads whose rows share 128-byte lines go to one XCD, whose L2 then reads them once (workgroups
    # go round the 8 XCDs): 34 sequences of 16 heads of 80 e4m3, 32.5 us without this and 25.5 with
    # it. Whole lines: 14 sequences of 16 heads of 128 bf16, 13.9 without and 14.8 with it.
    x = items + batch
    if dim * kc.size % 128:
        x = -(-x // 8) * 8
    launches = [("ek_paged_attention", (x, y), 64)]
    workspace = 0
    if most > _MIN_UNITS:              # some sequence may have more than one chunk
        workspace = (items + batch) * heads * (dim + 2) * 4 + batch * 8
        chunks = min(items, -(-most // _MIN_UNITS))
        # A wave per 16 chunks; where there are many sequences, few of them have many.
        waves = max(4, min(16, -(-chunks // 16), 4096 // (batch * heads)))
        launches.append(("ek_paged_attention_join", (batch, heads), 64 * waves))
    tail = _ATTEND.pack(
        qa.strides[0], qa.strides[1], oa.strides[0], oa.strides[1],
        *(s * kc.size for s in kc.strides[:3]), bt.strides[0], sl.strides[0], batch, heads,
        group, dim, kc.shape[1], kc.shape[0], capacity, window, *_page_division(kc.shape[1]),
        items, _MIN_UNITS, int(2 * kc.span() > _STREAM),
        0 if scale >= 0 else 0x80000000 if qa.kind == "fp32" else 0x80008000,
        # so small a scale is as good as none, and keeps -inf (no key there) what it is
        max(abs(scale) * k_scale * log2e, 2.0 ** -126), softcap * log2e, v_scale)
    if not workspace:
        tail = bytes(8) + tail         # the address of the partial results
    return _Plan("paged_attention.hip", macros, launches, arrays, {5, 6}, workspace, tail,
                 [(5, 0, True), (5, 1, False), (5, 2, False)]), out


# -- logits ----------------------------------------------------------------------------------

_LOGITS = struct.Struct("<12q3i4f4x")


MAX_BIASES = 1023                   # per row: 10 bits of a logit's word
MAX_HISTORY = (1 << 21) - 1         # per row: 21 bits


def _stretch(rows: int, vocab: int) -> int:
    """Logits per workgroup (of 512 threads): the longer stretch, which reads a history fewer
    times, unless that leaves CUs without a workgroup (256 x 128000 bf16, histories of up to 4096:
    44 us with 4096, 34 with 8192; one row of 32000 fp32, 20000 tokens: 6.0 and 6.9)."""
    return 4096 if rows * -(-vocab // 8192) < C.coarsen_cap() else 8192


def _per_row(name: str, x, rows: int, default: float):
    """(array or None, number) of a per-row setting given as a number or an array."""
    if x is None:
        return None, default
    if T.is_array_like(x):
        return _array(name, x, ("fp32",), 1, (rows,), dense=False), default
    return None, _f32(float(x))


def adjust_logits(logits, *, tokens=None, token_lens=None, prompt_lens=None,
                  repetition=None, frequency=None, presence=None, bias_ids=None, bias=None,
                  allowed=None, temperature=None, out=None):
    """Penalties for repeated tokens, biases, a temperature and a mask on rows of logits, in
    this order, computed in 32 bits (where 16-bit logits are divided, by the divisor's 32-bit
    reciprocal) and rounded once to their type:

    1. tokens that occur in the row's history: x / `repetition` where x > 0, else
       x * `repetition`;
    2. with c the number of times a token occurs in the generated part of the history:
       x - `frequency` * c, and - `presence` where c > 0;
    3. plus the sum of the row's biases for that token;
    4. divided by `temperature` where that is above 0;
    5. -inf where the token is not allowed, whatever the logit was. A row that allows none is
       -inf throughout.

    Args:
        logits: `[rows, vocabulary]`, float32, float16 or bfloat16.
        tokens: the history, int32 `[rows, length]`, shorter than 2^21; ids outside the
            vocabulary are ignored.
        token_lens: how much of each row of `tokens` counts, int32 `[rows]`; all without it.
        prompt_lens: how much of that is the prompt, int32 `[rows]`; none without it.
        repetition, frequency, presence, temperature: a number, or float32 `[rows]`
            (`repetition` from 2^-60 to 2^60).
        bias_ids, bias: int32 and float32 `[rows, entries]`, at most 1023 entries; ids outside
            the vocabulary are ignored, entries with the same id add up in their order.
        allowed: int32 `[rows, words]`, 32 tokens to a word: token t is bit t % 32 of word
            t // 32. One mask for all rows is an expanded array.
        out: where the result goes (`logits` itself will do); new without it.

    Returns:
        The adjusted logits, of the type of `logits`.
    """
    try:
        key = (2, logits.dtype, logits.shape, logits.stride(), logits.get_device(),
               *[x if x is None or x.__class__ in _NUMBERS else
                 (x.dtype, x.shape, x.stride(), x.get_device())
                 for x in (tokens, token_lens, prompt_lens, repetition, frequency, presence,
                           temperature, bias_ids, bias, allowed, out)])
        plan = _plans.get(key)
    except (AttributeError, TypeError, RuntimeError):
        key = plan = None              # arrays of another kind, or no arrays
    given = out is not None
    if plan is None:
        plan, out = _logits_plan(logits, tokens, token_lens, prompt_lens, repetition, frequency,
                                 presence, temperature, bias_ids, bias, allowed, out)
        if plan is None:
            return out
        _keep(key, plan)
    elif not given:
        out = _like(logits)
    arrays = [logits, out, tokens, token_lens, prompt_lens,
              *[None if x is None or x.__class__ in _NUMBERS or not
                (key is not None or T.is_array_like(x)) else x
                for x in (repetition, frequency, presence, temperature)],
              bias_ids, bias, allowed]
    if given:
        plan.check_apart(arrays)
    plan.run(arrays)
    return out


_NUMBERS = (float, int)


def _logits_plan(logits, tokens, token_lens, prompt_lens, repetition, frequency, presence,
                 temperature, bias_ids, bias, allowed, out):
    """The checked call's plan (None: nothing to do) and its `out`."""
    la = _array("logits", logits, ("fp32", "fp16", "bf16"), 2)
    rows, vocab = la.shape
    ta = tl = pl = None
    if tokens is not None:
        ta = _array("tokens", tokens, ("i32",), 2, (rows, None))
        if token_lens is not None:
            tl = _array("token_lens", token_lens, ("i32",), 1, (rows,), dense=False)
        if prompt_lens is not None:
            pl = _array("prompt_lens", prompt_lens, ("i32",), 1, (rows,), dense=False)
    else:
        _need(all(x is None for x in (token_lens, prompt_lens, repetition, frequency,
                                      presence)),
              "lengths and penalties need the history (`tokens`)")
    _need((bias_ids is None) == (bias is None), "`bias_ids` and `bias` go together")
    ia = ba = None
    if bias is not None:
        ia = _array("bias_ids", bias_ids, ("i32",), 2, (rows, None))
        ba = _array("bias", bias, ("fp32",), 2, ia.shape)
    aa = None
    if allowed is not None:
        aa = _array("allowed", allowed, ("i32",), 2, (rows, None))
        _need(aa.shape[1] * 32 >= vocab, f"`allowed` has {aa.shape[1]} words: {vocab} tokens "
                                         f"need {-(-vocab // 32)}")
    rep_a, rep = _per_row("repetition", repetition, rows, 1.0)
    freq_a, freq = _per_row("frequency", frequency, rows, 0.0)
    pres_a, pres = _per_row("presence", presence, rows, 0.0)
    temp_a, temp = _per_row("temperature", temperature, rows, 0.0)
    _positive("repetition", rep)
    # others lose digits, or all of them, as 32-bit numbers or in their reciprocals
    _need(temp <= 0 or 2.0 ** -126 <= temp <= 2.0 ** 126,
          f"`temperature` must be from 2^-126 to 2^126, or 0 for none, got {temp}")
    if out is None:
        out = T.new_empty(logits)
    oa = _array("out", out, (la.kind,), 2, la.shape)
    _written("out", oa)
    arrays = [("logits", la), ("out", oa), ("tokens", ta), ("token_lens", tl),
              ("prompt_lens", pl), ("repetition", rep_a), ("frequency", freq_a),
              ("presence", pres_a), ("temperature", temp_a), ("bias_ids", ia), ("bias", ba),
              ("allowed", aa)]
    _device_of(arrays)
    if rows == 0 or vocab == 0:
        return None, out
    _need(vocab < 1 << 30 and rows * -(-vocab // 4096) < 1 << 22,
          f"logits of shape {la.shape} are too large for one call")
    biases = ia.shape[1] if ia else 0
    _need(biases <= MAX_BIASES, f"at most {MAX_BIASES} biases of a row are supported, got "
                                f"{biases}")
    _need(ta is None or ta.shape[1] <= MAX_HISTORY,
          f"at most {MAX_HISTORY} tokens of history are supported, got "
          f"{ta.shape[1] if ta else 0}")
    n = _stretch(rows, vocab)
    macros = (("EK_Q", _Q[la.kind]), ("EK_N", n),
              ("EK_STREAM", int(rows * vocab * la.size > _STREAM_ROWS)))

    def step(a):
        return a.strides[0] if a is not None else 0

    tail = _LOGITS.pack(step(la), step(oa), step(ta), step(ia), step(ba), step(aa), step(tl),
                        step(pl), step(rep_a), step(freq_a), step(pres_a), step(temp_a), vocab,
                        ta.shape[1] if ta else 0, biases, rep, freq, pres, temp)
    return _Plan("adjust_logits.hip", macros,
                 [("ek_adjust_logits", (-(-vocab // n) * rows, 1), 512)], arrays, {1}, 0,
                 tail, [(1, 0, True)] + [(1, i, False) for i in range(2, 12)]), out


def specializations():
    """(source, macros) of the kernels that are worth compiling ahead."""
    for q, fp8 in ((2, 0), (1, 0), (0, 0), (2, 1), (1, 1)):
        for width in (64, 128, 256):
            for pad in (0, 1):
                size = 1 if fp8 else 2 if q else 4
                for keys in sorted({_step(width, size, short) for short in (False, True)}):
                    yield "paged_attention.hip", (("EK_Q", q), ("EK_FP8", fp8),
                                                  ("EK_DP", width), ("EK_PAD", pad),
                                                  ("EK_KT", keys))
        for pairs in (0, 1):
            for stream in (0, 1):
                yield "append_kv.hip", (("EK_Q", q), ("EK_FP8", fp8), ("EK_V", 8 if q else 4),
                                        ("EK_PAIRS", pairs), ("EK_STREAM", stream))
                for axes in (1, 2):
                    yield "append_kv.hip", (("EK_Q", q), ("EK_FP8", fp8),
                                            ("EK_V", 8 if q else 4), ("EK_PAIRS", pairs),
                                            ("EK_STREAM", stream), ("EK_AXES", axes))
    for q in (0, 1, 2):
        for n, stream in ((4096, 0), (8192, 0), (8192, 1)):
            yield "adjust_logits.hip", (("EK_Q", q), ("EK_N", n), ("EK_STREAM", stream))
