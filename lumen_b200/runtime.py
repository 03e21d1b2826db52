"""Host-side handles over the C ABI: fused kernels compiled from fusion bodies, GEMM, attention, scatter-add, launched
on device memory the caller holds. Tensors are duck-typed: the backend's own `lumen_b200.device.Tensor`, or any array
of another framework that answers `data_ptr()`, `shape`, `stride()` and `dtype` (a harness may pass torch CUDA
tensors; torch is never imported by this module unless the caller already did). Every kernel that runs is
liblumen_b200's."""

from __future__ import annotations

import ctypes
import math
import sys
import threading
from collections import OrderedDict

from lumen_b200 import _lib
from lumen_b200.graph import Graph


class _TorchDtypes(dict):
    """dtype name -> torch dtype, filled on first use so that importing this module does not import torch."""

    def __missing__(self, key):
        import torch

        self.update({
            "bool": torch.bool, "int8": torch.int8, "int16": torch.int16, "int32": torch.int32, "int64": torch.int64,
            "uint8": torch.uint8, "uint16": torch.uint16, "uint32": torch.uint32, "uint64": torch.uint64,
            "float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32, "float64": torch.float64,
        })  # fmt: skip
        return dict.__getitem__(self, key)


TORCH_DTYPES = _TorchDtypes()


_names: dict = {}  # dtype object -> lumen dtype name, as they are met


def dtype_name(dtype) -> str:
    """The lumen dtype name of a tensor's `dtype` attribute (a name already, or another framework's dtype object)."""
    if isinstance(dtype, str):
        return dtype
    name = _names.get(dtype)
    if name is None:
        name = str(dtype).rsplit(".", 1)[-1]  # "torch.bfloat16" -> "bfloat16"
        if name not in _lib.DTYPE_CODES:
            raise TypeError(f"no lumen dtype for {dtype!r}")
        _names[dtype] = name
    return name


_cuda_seen = False


def require_cuda() -> None:
    global _cuda_seen
    if not _cuda_seen:  # the devices of a process do not go away
        if _lib.lib().lb_device_count() <= 0:
            raise RuntimeError("lumen_b200 runs on a B200 GPU only: no CUDA device is available and there is no CPU fallback")
        _cuda_seen = True


def desc(t) -> _lib.LbTensor:
    """The lb_tensor descriptor of a device tensor (shape, element strides, data pointer)."""
    if not getattr(t, "is_cuda", True):
        raise ValueError("expected a CUDA tensor")
    return _lib.strided(t.data_ptr(), dtype_name(t.dtype), t.shape, t.stride())


_current = [0]


def set_current_stream(stream) -> None:
    """The stream launches go to when none is given and torch is not in the process (a `lumen_b200.device.Stream`)."""
    _current[0] = getattr(stream, "handle", stream) or 0


def current_stream() -> int:
    """The caller's current stream: torch's when the process uses torch (a harness), else the one set with
    `set_current_stream` (the legacy default stream by default)."""
    if _current[0] == 0:
        torch = sys.modules.get("torch")
        if torch is not None and torch.cuda.is_initialized():
            raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the handle without a Stream object around it
            return raw(torch.cuda.current_device()) if raw is not None else torch.cuda.current_stream().cuda_stream
    return _current[0]


def _stream(stream) -> int:
    return (current_stream() if stream is None else getattr(stream, "handle", stream)) or 0


class Fusion:
    """One generated kernel for a fusion body (`lb_fusion_compile` / `lb_fusion_launch`)."""

    def __init__(self, body: Graph | str):
        text = body if isinstance(body, str) else body.to_text()
        handle = ctypes.c_void_p()
        _lib.check(_lib.lib().lb_fusion_compile(text.encode(), ctypes.byref(handle)))
        self.handle = handle
        self.n_inputs = _lib.lib().lb_fusion_num_inputs(handle)
        self.n_outputs = _lib.lib().lb_fusion_num_outputs(handle)
        self.scratch_bytes = _lib.lib().lb_fusion_scratch_bytes(handle)
        self.body = body if isinstance(body, Graph) else None

    @property
    def source(self) -> str:
        return _lib.lib().lb_fusion_source(self.handle).decode()

    def launch_raw(self, descs, scratch_ptr=None, stream=None) -> None:
        arr = (_lib.LbTensor * len(descs))(*descs)
        _lib.check(
            _lib.lib().lb_fusion_launch(
                self.handle, arr, len(descs), scratch_ptr, current_stream() if stream is None else stream
            )
        )

    def __call__(self, *inputs, out=None, stream=None):
        """Runs the kernel on CUDA tensors; allocates the outputs unless `out` gives them."""
        require_cuda()
        if self.body is None:
            raise RuntimeError("calling a Fusion built from text needs explicit outputs: use launch_raw")
        if out is None:
            out = [_empty_like_input(inputs[0], self.body.types[v].shape, self.body.types[v].dtype) for v in self.body.outputs]
        # partial sums between the call's two kernels: another call must not meet them, on whatever stream, thread or device
        scratch = _workspace(inputs[0], (self.scratch_bytes,), "uint8", stream) if self.scratch_bytes else None
        self.launch_raw([desc(t) for t in (*inputs, *out)], scratch.data_ptr() if scratch is not None else None, stream)
        return out


_regions: dict = {}  # device -> its regions, as they were reserved


def _empty_like_input(like, shape, dtype: str):
    """A new dense device tensor of `shape`/`dtype` in the framework `like` comes from: torch for a torch tensor (the
    harness's convenience), else the backend's own regions of the current device (grown in 256 MiB reservations)."""
    if type(like).__module__.startswith("torch"):
        torch = sys.modules["torch"]
        if type(like) is torch.Tensor:  # 1.5 and 2.0 us a tensor, where `empty` takes 2.4 to read its arguments
            if like.shape == shape:
                return torch.empty_like(like, dtype=TORCH_DTYPES[dtype], memory_format=torch.contiguous_format)
            return like.new_empty(shape, dtype=TORCH_DTYPES[dtype])
        return torch.empty(shape, dtype=TORCH_DTYPES[dtype], device=like.device)
    from lumen_b200.device import ITEMSIZE, Region, current_device

    nbytes = max(math.prod(shape) * ITEMSIZE[dtype], 1)
    regions = _regions.setdefault(current_device(), [])
    for region in regions:
        try:
            return region.empty(shape, dtype)
        except _lib.LumenError:
            continue
    region = Region(max(nbytes + 4096, 256 << 20))
    regions.append(region)
    return region.empty(shape, dtype)


_workspaces: OrderedDict = OrderedDict()  # (device, stream) -> region, the latest used last
_workspaces_lock = threading.Lock()
_WORKSPACE_STREAMS = 8


def _workspace(like, shape, dtype: str, stream):
    """Memory of one call on `stream`, which may be dropped as soon as the call's kernels are queued: what the memory is given to next
    is queued on the same stream. From torch's allocator with `stream` current for a torch tensor, else from a region that serves
    this stream of the current device alone; the regions of the eight latest streams are kept (freeing one waits for its work)."""
    if type(like).__module__.startswith("torch"):
        if stream is None and _current[0] == 0:  # torch's current stream
            return _empty_like_input(like, shape, dtype)
        torch, handle = sys.modules["torch"], _stream(stream)
        with torch.cuda.stream(torch.cuda.ExternalStream(handle, like.device) if handle else torch.cuda.default_stream(like.device)):
            return _empty_like_input(like, shape, dtype)
    from lumen_b200.device import ITEMSIZE, Region, current_device

    key = (current_device(), _stream(stream))
    with _workspaces_lock:
        if key in _workspaces:
            _workspaces.move_to_end(key)
            try:
                return _workspaces[key].empty(shape, dtype)
            except _lib.LumenError:  # too small, or in use by other threads' calls: one that holds all of it takes its place
                live = _workspaces[key].stats()["live_bytes"]
        else:
            live = 0
        region = Region(max(live + math.prod(shape) * ITEMSIZE[dtype] + 4096, 32 << 20))
        work = region.empty(shape, dtype)  # (reserves the memory: a region that cannot be had takes no place)
        _workspaces[key] = region
        while len(_workspaces) > _WORKSPACE_STREAMS:
            _workspaces.popitem(last=False)
        return work


GEMM_KERNELS = {"auto": 0, "tcgen05": 1, "simt": 2, "tcgen05_1cta": 3}
EPILOGUES = {None: 0, "none": 0, "relu": 1, "add": 2, "mask_positive": 3}


def gemm(a, b, out, epilogue=None, kernel="auto", stream=None, scratch=None, aux=None):
    """`out[.., M, N] = a[.., M, K] @ b[.., K, N]` with float32 accumulation through `lb_gemm`. `a` and `b` may be
    transposed views (any unit-stride major); `out` is float32 or the operands' dtype, row-major. `scratch` (a
    uint8 tensor of `gemm_scratch_bytes` bytes) lets few-tile, long-K problems split K. Epilogues: "relu";
    "add" (`round(product) + aux`) and "mask_positive" (`aux > 0 ? round(product) : 0`) with `aux` shaped like `out`.
    Bit-identical from call to call; the same rows in a larger product may differ in the last bit (another number of K
    ranges, which depends on every dimension)."""
    require_cuda()
    scratch_ptr, scratch_bytes = (scratch.data_ptr(), scratch.numel() * scratch.element_size()) if scratch is not None else (0, 0)
    _lib.host().gemm(a, b, out, aux, EPILOGUES[epilogue], GEMM_KERNELS[kernel], scratch_ptr, scratch_bytes, _stream(stream))
    return out


def device_status() -> None:
    """Synchronises and raises if a kernel's bounded wait gave up (`lb_device_status`)."""
    _lib.check(_lib.lib().lb_device_status())


class _Torch:
    """What calls on plain torch tensors take from torch, looked up once: the lookups on the way to `_empty_like_input`, `_workspace` and
    `_stream` cost the host a microsecond a tensor, in front of kernels that take three."""

    tensor = None  # torch.Tensor, once such a tensor has been met

    @classmethod
    def takes(cls, t, stream) -> bool:
        """Whether `t` is a plain torch tensor and the call is for torch's current stream."""
        if cls.tensor is None and type(t).__module__.startswith("torch"):
            torch = sys.modules["torch"]
            if not hasattr(torch._C, "_cuda_getCurrentRawStream"):
                return False
            cls.empty_like, cls.dense, cls.float32, cls.bytes = torch.empty_like, torch.contiguous_format, torch.float32, torch.uint8
            cls.changed = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)
            cls.raw_stream, cls.device, cls.tensor = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice, torch.Tensor
        return type(t) is cls.tensor and stream is None and _current[0] == 0 and t.is_cuda

    @classmethod
    def like(cls, t):
        return cls.empty_like(t, memory_format=cls.dense)

    @classmethod
    def float32_like(cls, t):
        return cls.empty_like(t, dtype=cls.float32, memory_format=cls.dense)

    @classmethod
    def stream(cls) -> int:
        return cls.raw_stream(cls.device())


def attention_forward(q, k, v, scale=None, causal=False, out=None, lse=None, stream=None):
    """Flash attention forward through `lb_attention_fwd`: `q` [B, Sq, N, H], `k`/`v` [B, Sk, Nkv, H] bfloat16 views;
    returns `(o, lse)` with `o` [B, Sq, N, H] bfloat16 and `lse` [B, N, Sq] float32. Bit-identical from call to call; the
    same sequence in another batch may differ by a rounding of the probabilities to bfloat16 (another kernel, or another
    number of key ranges when few queries meet many keys)."""
    require_cuda()
    b, sq, n, h = q.shape
    sk = k.shape[1]
    if out is None and lse is None and _Torch.takes(q, stream):
        out, lse, handle = _Torch.like(q), q.new_empty((b, n, sq), dtype=_Torch.float32), _Torch.stream()
    else:
        if out is None:
            out = _empty_like_input(q, tuple(q.shape), dtype_name(q.dtype))
        if lse is None:
            lse = _empty_like_input(q, (b, n, sq), "float32")
        handle = _stream(stream)
    _lib.host().attention_fwd(float(scale if scale is not None else h**-0.5), bool(causal), sk - sq, q, k, v, out, lse, handle)
    return out, lse


# What the backward takes for dS whatever memory there is, and at most from a region, which is kept for its stream.
_SMALL_SCORES, _KEPT_SCORES = 64 << 20, 256 << 20


def _out_of_memory(error: RuntimeError) -> bool:
    if isinstance(error, _lib.LumenError):
        return "out of memory" in str(error)
    torch = sys.modules.get("torch")
    return torch is not None and isinstance(error, torch.OutOfMemoryError)


def _memory_is_short(t) -> bool:
    """Whether a request to torch's allocator for memory of `t`'s device has failed before: another one that does not fit would wait for the
    GPU and empty the allocator's cache once more. (10 us.)"""
    try:
        stats = sys.modules["torch"].cuda.memory_stats_as_nested_dict(t.device)
    except RuntimeError:  # an allocator that does not count
        return True
    return stats.get("num_alloc_retries", 0) + stats.get("num_ooms", 0) > 0


def _scores(q, nbytes: int, stream):
    """Memory for the dS that the backward hands on, or None where that may cost more than it gives."""
    if type(q).__module__.startswith("torch"):
        if nbytes > _SMALL_SCORES and _memory_is_short(q):
            return None
    elif nbytes > _KEPT_SCORES:
        return None
    try:
        return _workspace(q, (nbytes,), "uint8", stream)
    except RuntimeError as error:
        if not _out_of_memory(error):
            raise
        return None


def attention_backward(q, k, v, o, d_o, lse, scale=None, causal=False, delta=None, stream=None, deterministic=True, max_scratch=None):
    """Flash attention backward; returns `(dq, dk, dv)` shaped like `q`, `k`, `v`. `deterministic` (the default here)
    runs `lb_attention_bwd_scratch`, the dK/dV + dQ kernel pair that is bit-identical from run to run; without it
    `lb_attention_bwd_atomic` runs the reference backend's default mode, one kernel adding dQ atomically into a float32
    accumulator, at head dim 64, and the same pair elsewhere. At head dim 128 the pair hands dS on in memory of the call's, up to 4.5 GiB
    or `max_scratch` bytes (0: none), where there is such memory; the results are the same either way."""
    require_cuda()
    b, sq, n, h = q.shape
    sk = k.shape[1]
    plain = _Torch.takes(q, stream) and type(k) is type(v) is _Torch.tensor
    if plain:
        dq, dk, dv, handle = _Torch.like(q), _Torch.like(k), _Torch.like(v), _Torch.stream()
        if delta is None:
            delta = q.new_empty((b, n, sq), dtype=_Torch.float32)
    else:
        dq, dk, dv = (_empty_like_input(t, tuple(t.shape), dtype_name(t.dtype)) for t in (q, k, v))
        if delta is None:
            delta = _workspace(q, (b, n, sq), "float32", stream)
        handle = _stream(stream)
    dq_accum = _workspace(q, (b, sq, n, h), "float32", stream) if h == 64 and not deterministic else None
    scale, causal = float(scale if scale is not None else h**-0.5), bool(causal)
    nbytes = _lib.host().attention_bwd_scratch_bytes(scale, causal, sk - sq, q, k) if h == 128 else 0
    if max_scratch is not None:
        nbytes = max(0, min(nbytes, max_scratch))
    scores = _scores(q, nbytes, stream) if nbytes else None
    pointer, nbytes = (0, 0) if scores is None else (scores.data_ptr(), nbytes)
    _lib.host().attention_bwd(scale, causal, sk - sq, q, k, v, o, d_o, lse, delta, dq_accum, dq, dk, dv, pointer, nbytes, handle)
    return dq, dk, dv


def gemm_scratch_bytes(m: int, n: int, k: int, batch: int = 1) -> int:
    """Bytes of scratch with which `gemm` splits K for this problem (0: it would not split)."""
    return _lib.lib().lb_gemm_scratch_bytes(m, n, k, batch)


def scatter_add_rows(x, ids, updates, deterministic=True, stream=None):
    """`x` `[rows, width]` with `updates[t]` added into row `ids[t]` (clamped into range), through
    `lb_scatter_add_rows`. Deterministic form: a row hit more than once adds its updates in update order, rounding
    after each add, like the reference interpreter; otherwise float32 atomics in arrival order and one rounding."""
    require_cuda()
    lib = _lib.lib()
    lib.lb_scatter_add_scratch_bytes.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
    lib.lb_scatter_add_scratch_bytes.restype = ctypes.c_size_t
    T = ctypes.POINTER(_lib.LbTensor)
    lib.lb_scatter_add_rows.argtypes = [T, T, T, T, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_void_p]
    rows, width = x.shape
    nbytes = lib.lb_scatter_add_scratch_bytes(rows, width, ids.numel(), int(deterministic))
    scratch = _workspace(x, (max(nbytes, 4),), "uint8", stream)
    out = _empty_like_input(x, tuple(x.shape), dtype_name(x.dtype))
    updates = updates.reshape(-1, width)  # held until the kernels are queued: a view, or a copy of one with other strides
    dx, di, du, do = desc(x), desc(ids), desc(updates), desc(out)
    _lib.check(lib.lb_scatter_add_rows(ctypes.byref(dx), ctypes.byref(di), ctypes.byref(du), ctypes.byref(do), scratch.data_ptr(),
                                       nbytes, int(deterministic), current_stream() if stream is None else stream))
    return out


def _outputs(like, stream, *wanted):
    """New dense tensors of `(shape, dtype name)` each, None for None, and the handle of the stream."""
    if _Torch.takes(like, stream):
        return [None if w is None else like.new_empty(w[0], dtype=TORCH_DTYPES[w[1]]) for w in wanted], _Torch.stream()
    return [None if w is None else _empty_like_input(like, *w) for w in wanted], _stream(stream)


def _scratch(like, stream):
    """What the native path calls for a call's workspace: `nbytes` -> memory for the kernels queued on `stream` (see `_workspace`)."""
    if _Torch.takes(like, stream):
        return lambda nbytes: like.new_empty(nbytes, dtype=_Torch.bytes)
    return lambda nbytes: _workspace(like, (nbytes,), "uint8", stream)


def _results_like(tensors, out, stream):
    """`out`, or new dense tensors like each of `tensors`, and the handle of the stream."""
    if out is not None:
        return out, _stream(stream)
    if _Torch.takes(tensors[0], stream):
        try:
            return [_Torch.like(t) for t in tensors], _Torch.stream()
        except TypeError:  # one of them is another framework's
            pass
    return [_empty_like_input(t, tuple(t.shape), dtype_name(t.dtype)) for t in tensors], _stream(stream)


def _written(tensors):
    """Tells autograd that the caller's `tensors` have other values now, so that a backward pass that kept one of them raises as it does for torch's
    own in-place operations."""
    if len(tensors) and type(tensors[0]) is _Torch.tensor:
        try:
            return _Torch.changed(tensors)
        except RuntimeError:  # one of them is another framework's
            pass
    torch = sys.modules.get("torch")
    known = [t for t in tensors if isinstance(t, torch.Tensor)] if torch else ()
    if known:
        torch.autograd.graph.increment_version(known)


def qk_norm_rope(q, k, cos, sin, positions=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, out=None, stream=None):
    """Norms of queries and keys for each head and the position rotation, in one pass through `lb_qk_norm_rope`. `q` `[B, S, N, H]` and `k`
    `[B, S, Nkv, H]` are views of float16, bfloat16 or float32 (of a packed projection, say), H up to 256. Each head's row becomes
    `z = x / sqrt(mean(x^2) + eps) * weight`; then its first `2 * pairs` elements turn, `y_a = z_a cos - z_b sin`, `y_b = z_b cos + z_a sin`, in pairs
    `(i, i + pairs)`, or `(2i, 2i + 1)` with `interleaved`, by the float32 tables `cos` and `sin` `[positions, pairs]`. `positions`: int32 or int64,
    `[S]` or `[B, S]`, clamped into the tables; None is 0, 1, 2 ... Weights: `[H]` of `q`'s dtype or float32; None is all ones. Returns `(q, k)`
    of the operands' dtype, in `out` if given: `(q, k)` themselves, or memory that overlaps no tensor of the call. Bit-identical from call to call; the
    same rows among others may differ by a rounding."""
    require_cuda()
    (q_out, k_out), handle = _results_like((q, k), out, stream)
    _lib.host().qk_norm_rope(eps, bool(interleaved), q, k, cos, sin, positions, q_weight, k_weight, q_out, k_out, handle)
    if out is not None:
        _written((q_out, k_out))
    return q_out, k_out


def qk_norm_rope_backward(d_q_out, d_k_out, q, k, cos, sin, positions=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, out=None,
                          stream=None):
    """The backward pass of `qk_norm_rope` on the same operands: returns `(d_q, d_k, d_q_weight, d_k_weight)`, the last two of their weight's dtype and
    None without one. `out` takes `d_q` and `d_k`, which may be `(d_q_out, d_k_out)` or memory that overlaps no tensor of the call. Bit-identical from
    call to call."""
    require_cuda()
    (d_q, d_k), handle = _results_like((q, k), out, stream)
    weights = [w for w in (q_weight, k_weight) if w is not None]
    grads = _results_like(weights, None, stream)[0] if weights else []
    d_q_weight, d_k_weight = grads.pop(0) if q_weight is not None else None, grads.pop() if k_weight is not None else None
    _lib.host().qk_norm_rope_bwd(eps, bool(interleaved), d_q_out, d_k_out, q, k, cos, sin, positions, q_weight, k_weight, d_q, d_k, d_q_weight, d_k_weight,
                                 _scratch(q, stream), handle)
    if out is not None:
        _written((d_q, d_k))
    return d_q, d_k, d_q_weight, d_k_weight


ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}


def _activation(name) -> int:
    if name not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {name!r}")
    return ACTIVATIONS[name]


def gated_mlp_forward(x, w_gate_up, w_down, activation="silu", residual=None, save=True, stream=None):
    """The gated feed-forward block through `lb_gated_mlp_fwd`: `y = (f(x Wg^T) * (x Wu^T)) Wd^T` for the rows of `x` `[.., D]`, with `w_gate_up`
    `[2 F, D]` (the F rows of Wg, then those of Wu), `w_down` `[D, F]` and `f` "silu", "gelu" (its tanh form) or "relu". Returns `(y, gate_up, h)`:
    `gate_up` `[.., 2 F]`, the two projections (None with `save=False`), and `h` `[.., F]`, their gated product, are what the backward pass
    reads. Sums are float32, and `h` is computed from them. `residual` (16-bit dtypes, shaped like `y`) is added to the rounded product. float16,
    bfloat16 or float32; the tensor cores take 16-bit operands whose rows are 16-byte aligned, the CUDA cores the others. Bit-identical from call to
    call; the same rows among others may differ by a rounding."""
    require_cuda()
    act, lead, f = _activation(activation), x.shape[:-1], w_gate_up.shape[0] // 2
    if _Torch.takes(x, stream):
        y, gate_up, h, handle = _Torch.like(x), x.new_empty((*lead, 2 * f)) if save else None, x.new_empty((*lead, f)), _Torch.stream()
    else:
        dtype = dtype_name(x.dtype)
        (y, gate_up, h), handle = _outputs(x, stream, (tuple(x.shape), dtype), ((*lead, 2 * f), dtype) if save else None, ((*lead, f), dtype))
    _lib.host().gated_mlp_fwd(act, x, w_gate_up, w_down, residual, y, gate_up, h, _scratch(x, stream), handle)
    return y, gate_up, h


def gated_mlp_backward(d_y, x, w_gate_up, w_down, gate_up, h, activation="silu", stream=None):
    """The backward pass of `gated_mlp_forward` through `lb_gated_mlp_bwd`: returns `(d_x, d_w_gate_up, d_w_down)` of the operands' dtype. (A residual's
    gradient is `d_y` itself.) Bit-identical from call to call."""
    require_cuda()
    act = _activation(activation)
    (d_x, d_wgu, d_wd), handle = _results_like((x, w_gate_up, w_down), None, stream)
    _lib.host().gated_mlp_bwd(act, d_y, x, w_gate_up, w_down, gate_up, h, d_x, d_wgu, d_wd, _scratch(x, stream), handle)
    return d_x, d_wgu, d_wd


def _norm(tensors, out, max_norm, like, stream):
    require_cuda()
    tensors, out = (t if t is None or type(t) in (list, tuple) else list(t) for t in (tensors, out))
    if like is None:
        if len(tensors) == 0:
            raise ValueError("the norm of no tensors needs `like`, a tensor on the GPU")
        like = tensors[0]
    (norm,), handle = _outputs(like, stream, ((), "float32"))
    _lib.host().clip_grad_norm(tensors, out, max_norm, norm, _scratch(like, stream), handle)
    if max_norm is not None:
        _written(tensors if out is None else out)
    return norm


def grad_norm(tensors, like=None, stream=None):
    """The 2-norm of all elements of a list of tensors (float16, bfloat16 and float32 in any mix; each dense, in any order of its dimensions), as a
    0-d float32 tensor on the device, through `lb_grad_norm`. A tensor listed twice counts twice. `like` says where the result goes if the list may
    be empty. The sum of squares is held in 64 bits; the same bits from call to call."""
    return _norm(tensors, None, None, like, stream)


def clip_grad_norm(tensors, max_norm, out=None, like=None, stream=None):
    """`grad_norm`, and every tensor times `min(1, max_norm / (norm + 1e-6))`: in place, or into `out`, a list of tensors of the same dtypes and
    layouts that share no memory with one another or with `tensors`. `max_norm` is finite (`grad_norm` is the norm alone). Returns the norm before
    clipping (0-d float32, on the device); nothing waits for it. In place, tensors of a norm within the bound are read once and left alone. An infinite or NaN norm makes every tensor 0 or NaN, as
    the quotient says."""
    return _norm(tensors, out, float(max_norm), like, stream)


REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _reduction(name) -> int:
    if name not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {sorted(REDUCTIONS)}, got {name!r}")
    return REDUCTIONS[name]


def linear_cross_entropy(x, weight, targets, reduction="mean", ignore_index=-100, stream=None):
    """Softmax cross entropy of the projection `x @ weight^T` through `lb_linear_cross_entropy`, without the logits ever being in memory as a whole: `x`
    `[.., D]` (hidden states), `weight` `[V, D]` (an output head), `targets` `[..]` int32 or int64. Returns `(loss, lse)`: the loss of each row, or its
    sum or mean over the rows that count (0 where none does), and each row's log-sum-exp, which the backward pass reads; both float32. A row whose target
    is `ignore_index` does not count; other targets are clamped into the vocabulary. float16, bfloat16 or float32. Infinities and NaN in a row that counts
    are in its loss, as the formula has them, whatever the type. Bit-identical from call to call; the same rows among others may differ by a rounding."""
    require_cuda()
    code = _reduction(reduction)
    if _Torch.takes(x, stream) and type(targets) is _Torch.tensor:
        lse, handle = _Torch.float32_like(targets), _Torch.stream()
        loss = x.new_empty((), dtype=_Torch.float32) if code else _Torch.float32_like(targets)
    else:
        shape = tuple(targets.shape)
        (loss, lse), handle = _outputs(x, stream, (() if code else shape, "float32"), (shape, "float32"))
    _lib.host().linear_cross_entropy(code, ignore_index, x, weight, targets, loss, lse, _scratch(x, stream), handle)
    return loss, lse


def linear_cross_entropy_backward(d_loss, x, weight, targets, lse, reduction="mean", ignore_index=-100, stream=None):
    """The backward pass of `linear_cross_entropy` on the same operands, through `lb_linear_cross_entropy_bwd`: returns `(d_x, d_weight)` of the
    operands' shapes and dtype. `d_loss` is the gradient of the loss, float32 of its shape (None: ones). The logits are computed anew, a piece of the
    vocabulary at a time. Rows that do not count have a gradient of zero and no part in `d_weight`, whatever stands in them. Bit-identical from call to
    call."""
    require_cuda()
    code = _reduction(reduction)
    (d_x, d_weight), handle = _results_like((x, weight), None, stream)
    _lib.host().linear_cross_entropy_bwd(code, ignore_index, d_loss, x, weight, targets, lse, d_x, d_weight, _scratch(x, stream), handle)
    return d_x, d_weight


ADAMW_BLOCK = 256  # elements that share a scale where moments are held in 8 bits


def adamw_state(params, bits=32):
    """The moments of a first `adamw_step` on `params`: `(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale)`, lists of zeros. With `bits=32` the
    moments are float32 tensors shaped like the parameters and there are no scales (None); with `bits=8` they are uint8 tensors of e4m3 codes, with a
    float32 scale for each 256 elements."""
    if bits not in (8, 32):
        raise ValueError(f"bits must be 8 or 32, got {bits!r}")
    params = list(params)

    def zeros(dtype, shape=None):
        return [_zeros_like_input(t, None if shape is None else shape(t), dtype) for t in params]

    if bits == 32:
        return zeros("float32"), zeros("float32"), None, None

    def blocks(t):
        return (-(-math.prod(t.shape) // ADAMW_BLOCK),)

    return zeros("uint8"), zeros("uint8"), zeros("float32", blocks), zeros("float32", blocks)


def _zeros_like_input(like, shape, dtype: str):
    """Zeros in the framework `like` comes from, of its shape and layout unless `shape` is given."""
    if type(like).__module__.startswith("torch"):
        torch = sys.modules["torch"]
        like = like.detach()
        return torch.zeros_like(like, dtype=TORCH_DTYPES[dtype]) if shape is None else torch.zeros(shape, dtype=TORCH_DTYPES[dtype], device=like.device)
    out = _empty_like_input(like, tuple(like.shape) if shape is None else shape, dtype)
    _lib.check(out.lib.lb_fill_bytes(out.ptr, 0, out.nbytes, current_stream()))
    return out


def adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, exp_avg_scale=None, exp_avg_sq_scale=None,
               masters=None, norm=None, max_norm=None, stream=None):
    """One AdamW step over a list of parameters through `lb_adamw_step`, in place: with `m` and `v` the moments of the gradient and of its square,
    `w (1 - lr weight_decay) - lr (m / (1 - b1^step)) / (sqrt(v / (1 - b2^step)) + eps)` in float32, rounded once to the parameter's type. Parameters of
    float16, bfloat16 and float32 in any mix, dense in any order of their dimensions; gradients of the same type or float32. `exp_avg` and `exp_avg_sq` are
    float32 tensors of the parameters' layout, or, with their scales, moments in 8 bits (`adamw_state` makes both; one that is not finite takes its block of 256
    with it). `masters`: float32 copies of 16-bit
    parameters, on which the step is then taken (None in the place of a parameter that has none). `step` counts from 1; it and `lr` are numbers or one-element
    tensors on the device (int32, int64 or float32; float32), which a captured graph reads anew in every replay. With `norm` (what `grad_norm` gives) and
    `max_norm` the gradients are taken times `min(1, max_norm / (norm + 1e-6))`, as `clip_grad_norm` would leave them, and stay as they are. Nothing waits
    for the device. The same bits from call to call."""
    require_cuda()
    params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, masters = (
        t if t is None or type(t) in (list, tuple) else list(t) for t in (params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, masters))  # fmt: skip
    if (norm is None) != (max_norm is None):
        raise ValueError("clipping needs both the norm and max_norm")
    if not len(params):
        return
    handle = _Torch.stream() if _Torch.takes(params[0], stream) else _stream(stream)
    _lib.host().adamw_step(params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, masters, step, lr, *betas, eps, weight_decay, norm,
                           0.0 if max_norm is None else max_norm, handle)  # fmt: skip
    changed = [*params, *exp_avg, *exp_avg_sq]
    if exp_avg_scale:
        changed += [*exp_avg_scale, *exp_avg_sq_scale]
    if masters:
        changed += [t for t in masters if t is not None]
    _written(changed)
