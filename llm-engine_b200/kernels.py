"""Device-side operators of the paged-KV path, named and shaped after llm-engine's
launchers (include/engine/cuda_kernels.h:43-62) and called through the C ABI.

Arguments are torch CUDA tensors (torch is used only for device memory and
streams); element type is taken from the tensors: float16 (the reference's CUDA
dtype), bfloat16 or float32.  Errors raise, as the reference launchers throw; there
is no CPU path.
"""
from __future__ import annotations

import contextlib
import ctypes as C

from . import _lib

_SUFFIX = {"torch.float16": "f16", "torch.bfloat16": "bf16", "torch.float32": "f32"}


def _suffix(t) -> str:
    try:
        return _SUFFIX[str(t.dtype)]
    except KeyError:
        raise TypeError(f"unsupported KV element type {t.dtype}") from None


_BY_DTYPE = {}      # (entry point, torch.dtype) -> (name, function): the names are put together once


def _fn(op: str, t):
    """(name, C function) of the entry point `op` for the element type of pool tensor t."""
    found = _BY_DTYPE.get((op, t.dtype))
    if found is None:
        name = op + _suffix(t)
        found = _BY_DTYPE[op, t.dtype] = (name, getattr(_lib.lib(), name))
    return found


def _ptr(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("paged-KV operators take CUDA tensors; there is no CPU path")
    if not t.is_contiguous():
        raise ValueError("paged-KV operators take contiguous tensors")
    return t.data_ptr()


def _no_raw_stream(_):
    import torch
    return torch.cuda.current_stream().cuda_stream


_raw_stream = None   # (device index) -> the current stream's handle


def _stream(stream):
    """The stream's handle; None: the current stream of the current device.  A torch.cuda.Stream object is not
    built for it: that alone takes 3.4 us, as long as a launch."""
    global _raw_stream
    if stream is not None:
        return getattr(stream, "cuda_stream", stream)
    import torch
    if _raw_stream is None:
        torch.cuda.init()
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _no_raw_stream)
    return _raw_stream(torch.cuda.current_device())


def launch_store_kv(k, v, slots, k_cache, v_cache, n_tokens: int, kv_dim: int, stream=None) -> None:
    """k_cache[slots[t]] = k[t], v_cache[slots[t]] = v[t] (engine::launch_store_kv)."""
    fn, call = _fn("pkv_append_", k_cache)
    st = call(_ptr(k), _ptr(v), _ptr(slots), _ptr(k_cache), _ptr(v_cache), n_tokens, kv_dim,
              _stream(stream))
    _lib.check(fn, st)


def launch_rope_store_kv(q, k, v, positions, cos_table, sin_table, slots, k_cache, v_cache, n_tokens: int,
                         q_heads: int, kv_heads: int, head_dim: int, stream=None) -> None:
    """launch_rope(q) + launch_rope(k) + launch_store_kv in one pass: q rotated in place, rotated k and v
    written to their slots (cos/sin: fp32 tables [max_positions][head_dim/2])."""
    fn, call = _fn("pkv_rope_append_", k_cache)
    st = call(_ptr(q), _ptr(k), _ptr(v), _ptr(positions), _ptr(cos_table), _ptr(sin_table),
              _ptr(slots), _ptr(k_cache), _ptr(v_cache), n_tokens, q_heads, kv_heads, head_dim,
              _stream(stream))
    _lib.check(fn, st)


# The checks below run once per call and layer: a few tenths of a microsecond per tensor, attributes looked up once.
def _wrong(tensors, dtype, device: int, what: str, rows: bool = False):
    """Raises the error of the first of `tensors` that is not a contiguous (or `rows`) `dtype` tensor of CUDA device `device`."""
    for t in tensors:
        if not t.is_cuda:
            raise ValueError("paged-KV operators take CUDA tensors; there is no CPU path")
        if t.dtype is not dtype:
            raise TypeError(f"{what} must be {dtype}, not {t.dtype}")
        if t.get_device() != device:
            raise ValueError(f"{what} lie on different devices: {t.get_device()} and {device}")
        if not rows and not t.is_contiguous():
            raise ValueError("paged-KV operators take contiguous tensors")


def _check(tensors, dtype, device: int, what: str) -> None:
    for t in tensors:
        if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous():
            _wrong(tensors, dtype, device, what)


def _rows(t, cols: int, n_rows: int, what: str):
    """(pointer, elements from one row to the next) of a [rows][cols] tensor whose rows may lie apart."""
    shape, stride = t.shape, t.stride()      # (size(0) and stride(0) take twice as long)
    if len(shape) != 2 or shape[1] != cols or shape[0] < n_rows or (stride[1] != 1 and cols > 1):
        raise ValueError(f"{what} must be [at least {n_rows}][{cols}] with contiguous rows, not {tuple(shape)} with strides {stride}")
    return t.data_ptr(), stride[0]


_torch = None
_one_device = False


def _this_device(device: int):
    """None if `device` is current, else a context in which it is (launches follow the current one)."""
    global _torch, _one_device
    if _torch is None:
        import torch
        _torch, _one_device = torch, torch.cuda.device_count() == 1
        _stream(None)
    return None if _one_device or _torch.cuda.current_device() == device else _torch.cuda.device(device)


def _stream_of(stream, device: int):
    """_stream for a device that is the current one."""
    return _raw_stream(device) if stream is None else getattr(stream, "cuda_stream", stream)


def launch_qk_norm_rope_store_kv(q, k, v, q_weight, k_weight, eps: float, positions, cos_table, sin_table, slots, q_out, k_cache,
                                 v_cache, n_tokens: int, q_heads: int, kv_heads: int, head_dim: int, stream=None) -> None:
    """launch_rope_store_kv for models that norm the heads of q and k first: RMS norm per head with its weight,
    rotation, append, in one pass.  q, k and v are [rows][heads*head_dim] and may be column ranges of one
    projection's output; q_out (contiguous) receives the rotated q.  Rows whose position is outside the tables are
    left alone, rows whose slot is outside the pools bring no K/V (padded steps)."""
    device, dtype = k_cache.get_device(), k_cache.dtype
    if device < 0:
        _wrong((k_cache,), dtype, device, "pools")
    other = _this_device(device)
    if other is not None:
        with other:
            return launch_qk_norm_rope_store_kv(q, k, v, q_weight, k_weight, eps, positions, cos_table, sin_table, slots, q_out, k_cache,
                                                v_cache, n_tokens, q_heads, kv_heads, head_dim, stream)
    q_dim, kv_dim = q_heads * head_dim, kv_heads * head_dim
    i32, f32 = _torch.int32, _torch.float32
    if not (q.dtype is dtype and k.dtype is dtype and v.dtype is dtype and q_weight.dtype is dtype and k_weight.dtype is dtype
            and q_out.dtype is dtype and v_cache.dtype is dtype and positions.dtype is i32 and slots.dtype is i32
            and cos_table.dtype is f32 and sin_table.dtype is f32
            and device == q.get_device() == k.get_device() == v.get_device() == q_weight.get_device() == k_weight.get_device()
            == positions.get_device() == cos_table.get_device() == sin_table.get_device() == slots.get_device()
            == q_out.get_device() == v_cache.get_device()
            and q_weight.is_contiguous() and k_weight.is_contiguous() and positions.is_contiguous() and cos_table.is_contiguous()
            and sin_table.is_contiguous() and slots.is_contiguous() and q_out.is_contiguous() and k_cache.is_contiguous()
            and v_cache.is_contiguous()):
        _wrong((q_weight, k_weight, q_out, k_cache, v_cache), dtype, device, "weights, q_out and pools")
        _wrong((positions, slots), i32, device, "positions and slots")
        _wrong((cos_table, sin_table), f32, device, "cos and sin tables")
        _wrong((q, k, v), dtype, device, "q, k and v", rows=True)
    tables, n_pool = cos_table.shape, k_cache.numel()
    if tables != sin_table.shape or len(tables) != 2 or 2 * tables[1] != head_dim:
        raise ValueError(f"cos and sin tables must both be [positions][{head_dim // 2}]")
    if q_weight.numel() != head_dim or k_weight.numel() != head_dim:
        raise ValueError(f"norm weights must have head_dim = {head_dim} elements")
    if positions.numel() < n_tokens or slots.numel() < n_tokens or q_out.numel() < n_tokens * q_dim:
        raise ValueError(f"fewer rows than n_tokens = {n_tokens}")
    if v_cache.numel() != n_pool:
        raise ValueError("K and V pools differ in size")
    fn, call = _fn("pkv_qk_norm_rope_append_", k_cache)
    qp, qs = _rows(q, q_dim, n_tokens, "q")
    kp, ks = _rows(k, kv_dim, n_tokens, "k")
    vp, vs = _rows(v, kv_dim, n_tokens, "v")
    st = call(qp, kp, vp, qs, ks, vs, q_weight.data_ptr(), k_weight.data_ptr(), eps, positions.data_ptr(), cos_table.data_ptr(),
              sin_table.data_ptr(), tables[0], slots.data_ptr(), q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
              n_pool // max(kv_dim, 1), n_tokens, q_heads, kv_heads, head_dim, _stream_of(stream, device))
    if st:
        _lib.check(fn, st)


def decode_workspace_bytes(n_tokens: int, q_heads: int, kv_heads: int, head_dim: int) -> int:
    return int(_lib.lib().pkv_decode_workspace_bytes(n_tokens, q_heads, kv_heads, head_dim))


def alloc_decode_workspace(n_tokens: int, q_heads: int, kv_heads: int, head_dim: int, device="cuda"):
    """A uint8 CUDA tensor large enough for split-K at this step size (256-byte aligned)."""
    import torch
    n = decode_workspace_bytes(n_tokens, q_heads, kv_heads, head_dim)
    return torch.empty(max(n, 256), dtype=torch.uint8, device=device)


def launch_attention_decode(q, k_cache, v_cache, block_tables, table_offset, token_seq, token_pos, out,
                            n_tokens: int, q_heads: int, kv_heads: int, head_dim: int, block_size: int,
                            scale: float, stream=None, workspace=None) -> None:
    """engine::launch_attention_decode; `workspace` (uint8 CUDA tensor) enables split-K."""
    fn, call = _fn("pkv_decode_attn_", k_cache)
    ws_ptr = _ptr(workspace)
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    st = call(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables), _ptr(table_offset),
              _ptr(token_seq), _ptr(token_pos), _ptr(out), n_tokens, q_heads, kv_heads,
              head_dim, block_size, C.c_float(scale), ws_ptr, ws_bytes, _stream(stream))
    _lib.check(fn, st)


def mixed_workspace_bytes(n_tokens: int, q_heads: int, kv_heads: int, head_dim: int) -> int:
    return int(_lib.lib().pkv_mixed_attn_workspace_bytes(n_tokens, q_heads, kv_heads, head_dim))


def launch_attention_mixed(q, k_cache, v_cache, block_tables, table_offset, token_seq, token_pos, out,
                           n_tokens: int, q_heads: int, kv_heads: int, head_dim: int, block_size: int,
                           scale: float, workspace, num_blocks: int = 0, min_run: int = 0, stream=None) -> None:
    """One call for a step that packs prefill chunks and decode tokens together, the way
    llm-engine's forward pass calls launch_attention_decode (src/model/cuda/cuda_model.cu:362-377):
    runs of at least min_run consecutive tokens of one sequence go to the tensor-core prefill kernel,
    the rest to the decode kernels; the split is made on the device."""
    fn, call = _fn("pkv_mixed_attn_", k_cache)
    st = call(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables), _ptr(table_offset),
              _ptr(token_seq), _ptr(token_pos), _ptr(out), n_tokens, q_heads, kv_heads, head_dim,
              block_size, num_blocks, C.c_float(scale), min_run, _ptr(workspace),
              workspace.numel() * workspace.element_size(), _stream(stream))
    _lib.check(fn, st)


# llm-engine keeps two names for the same operation, chosen by ENGINE_ATTN
# (src/model/cuda/cuda_model.cu:554-557); both are one kernel here.
launch_attention_decode_gqa = launch_attention_decode


def _passed(event, wait: bool) -> bool:
    """Whether the GPU has come past `event`, inside a stream capture too (torch's own query ends one)."""
    return bool(_lib.check("pkv_event_passed", _lib.lib().pkv_event_passed(event.cuda_event, wait)))


def _mark(event, stream, device: int):
    """`event`, recorded behind what `stream` (None, a stream or its handle) of the current device holds so far; what a stream that is being
    captured holds runs with the graph only, and the event stays where it was."""
    import torch
    if stream is not None and not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
    with contextlib.nullcontext() if stream is None else torch.cuda.stream(stream):
        if not torch.cuda.is_current_stream_capturing():
            event = event or torch.cuda.Event()
            event.record()
    return event


class _Staging:
    """Pinned memory that a plan is written to on the host and uploaded from.  A stream runs the upload when it gets there, perhaps
    after the next step's lengths are known or the plan object is gone, and torch's allocator does not know of it: until then the bytes
    are neither written again (writable) nor given back (the owner may drop them at any time)."""
    _left = []      # (event, bytes) whose owners are gone

    def __init__(self, n: int):
        import torch
        pending = []
        while _Staging._left:
            try:
                left = _Staging._left.pop()          # (one thread's at a time)
            except IndexError:
                break
            if not _passed(left[0], False):
                pending.append(left)
        _Staging._left.extend(pending)
        self.bytes = torch.empty(max(n, 256), dtype=torch.uint8, pin_memory=torch.cuda.is_available())
        self._sent = None

    def writable(self) -> None:
        if self._sent is not None:
            _passed(self._sent, True)

    def sent(self, stream, device: int) -> None:
        self._sent = _mark(self._sent, stream, device)

    def __del__(self, left=_left):
        if getattr(self, "_sent", None) is not None:
            left.append((self._sent, self.bytes))


class DecodePlan:
    """Split-K work list built once per step and shared by every layer's attention call."""

    def __init__(self, n_tokens: int, q_heads: int, kv_heads: int, head_dim: int, workspace=None, device="cuda",
                 num_blocks: int = 0):
        """num_blocks: blocks per K/V pool, if known: the kernels' tensor maps then end at the pool
        (a wrong block id reads zeros); 0 = unknown, as through llm-engine's own launcher signature."""
        import torch
        self.n_tokens, self.q_heads, self.kv_heads, self.head_dim = n_tokens, q_heads, kv_heads, head_dim
        self.num_blocks = num_blocks
        self.workspace = workspace if workspace is not None else alloc_decode_workspace(
            n_tokens, q_heads, kv_heads, head_dim, device)
        self._staging = _Staging(int(_lib.lib().pkv_decode_plan_staging_bytes(n_tokens, kv_heads)))
        self.staging = self._staging.bytes
        self.plan = _lib.DecodePlan()

    def _ws(self):
        return self.workspace.data_ptr(), self.workspace.numel()

    def build_host(self, token_pos_host, stream=None) -> "DecodePlan":
        """token_pos_host: int32 numpy array or CPU tensor of the packed tokens' positions."""
        import numpy as np
        pos = np.ascontiguousarray(token_pos_host, dtype=np.int32)
        p, n = self._ws()
        self._staging.writable()
        st = _lib.lib().pkv_decode_plan_host(pos.ctypes.data, self.n_tokens, self.q_heads, self.kv_heads,
                                             self.head_dim, self.staging.data_ptr(), self.staging.numel(), p, n,
                                             _stream(stream), C.byref(self.plan))
        self._staging.sent(stream, self.workspace.get_device())
        _lib.check("pkv_decode_plan_host", st)
        self.plan.num_blocks = self.num_blocks
        return self

    def build_host_image(self, token_pos_host) -> int:
        """The host planner without the upload: the image goes to self.staging (pinned) and its size
        is returned; the caller copies it to the start of self.workspace, typically as a node of a
        captured graph that is replayed every step."""
        import numpy as np
        pos = np.ascontiguousarray(token_pos_host, dtype=np.int32)
        n = C.c_size_t(0)
        self._staging.writable()
        st = _lib.lib().pkv_decode_plan_host_image(pos.ctypes.data, self.n_tokens, self.q_heads, self.kv_heads, self.head_dim,
                                                   self.staging.data_ptr(), self.staging.numel(), self.workspace.numel(),
                                                   C.byref(self.plan), C.byref(n))
        _lib.check("pkv_decode_plan_host_image", st)
        self.plan.num_blocks = self.num_blocks
        return int(n.value)

    def build_host_shared(self, idx, block_size: int, min_saved_bytes: int = -1, stream=None) -> "DecodePlan":
        """Shared-prefix-aware plan from the host copies of the step's index arrays (`idx`: a
        StepIndices as returned by pack_step): sequences whose tables start with the same blocks
        have that range read once per group of up to four tokens, if that saves at least
        min_saved_bytes of K/V reads per layer (-1: the library's default; 0: always)."""
        import numpy as np
        pos = np.ascontiguousarray(idx.token_pos, dtype=np.int32)
        seq = np.ascontiguousarray(idx.token_seq, dtype=np.int32)
        tabs = np.ascontiguousarray(idx.block_tables, dtype=np.int32)
        off = np.ascontiguousarray(idx.table_offset, dtype=np.int32)
        p, n = self._ws()
        self._staging.writable()
        st = _lib.lib().pkv_decode_plan_host_shared(pos.ctypes.data, seq.ctypes.data, tabs.ctypes.data, off.ctypes.data,
                                                    self.n_tokens, off.size, tabs.size, block_size, self.q_heads,
                                                    self.kv_heads, self.head_dim, min_saved_bytes, self.staging.data_ptr(),
                                                    self.staging.numel(), p, n, _stream(stream), C.byref(self.plan))
        self._staging.sent(stream, self.workspace.get_device())
        _lib.check("pkv_decode_plan_host_shared", st)
        self.plan.num_blocks = self.num_blocks
        return self

    @property
    def n_shared_units(self) -> int:
        return int(self.plan.reserved) >> 1

    def build_device(self, token_pos, stream=None) -> "DecodePlan":
        p, n = self._ws()
        st = _lib.lib().pkv_decode_plan_device(_ptr(token_pos), self.n_tokens, self.q_heads, self.kv_heads,
                                               self.head_dim, p, n, _stream(stream), C.byref(self.plan))
        _lib.check("pkv_decode_plan_device", st)
        self.plan.num_blocks = self.num_blocks
        return self

    def attention(self, q, k_cache, v_cache, block_tables, table_offset, token_seq, token_pos, out,
                  block_size: int, scale: float, stream=None) -> None:
        fn, call = _fn("pkv_decode_attn_planned_", k_cache)
        p, n = self._ws()
        st = call(C.byref(self.plan), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables),
                  _ptr(table_offset), _ptr(token_seq), _ptr(token_pos), _ptr(out), block_size,
                  C.c_float(scale), p, n, _stream(stream))
        _lib.check(fn, st)

    def append_attention(self, q, k, v, slots, k_cache, v_cache, block_tables, table_offset, token_seq, token_pos, out,
                         block_size: int, scale: float, stream=None) -> None:
        """launch_store_kv + attention in one chain (decode steps only: one token per sequence)."""
        fn, call = _fn("pkv_append_decode_attn_planned_", k_cache)
        p, n = self._ws()
        st = call(C.byref(self.plan), _ptr(q), _ptr(k), _ptr(v), _ptr(slots), _ptr(k_cache), _ptr(v_cache),
                  _ptr(block_tables), _ptr(table_offset), _ptr(token_seq), _ptr(token_pos), _ptr(out),
                  block_size, C.c_float(scale), p, n, _stream(stream))
        _lib.check(fn, st)


def _int32(a):
    """`a` as a contiguous int32 array; what would come out as other numbers (2^32 + 5 as 5, 1.5 as 1) is refused."""
    import numpy as np
    given = np.asarray(a)
    if given.dtype.kind in "iubf":
        with np.errstate(invalid="ignore"):
            out = np.ascontiguousarray(given, dtype=np.int32)
        if given.dtype == np.int32 or np.array_equal(out, given):
            return out
    raise ValueError("lengths and positions must be whole numbers of 32 bits")


class _SegmentPlan:
    """Work list of attention in which many rows see the same keys, built once per step on the host and used by
    every layer's call (include/pkv.h, pkv_segment_plan).  Its calls share one workspace: those that may
    overlap on the GPU need a plan each.  A plan may be made anew, or dropped, while the GPU still works on earlier calls; a graph
    that captured its calls needs it for as long as it is replayed."""

    def __init__(self, workspace_bytes, n_tokens: int, q_heads: int, kv_heads: int, head_dim: int, block_size: int, dtype,
                 num_blocks: int, workspace, device):
        import torch
        if str(dtype) not in _SUFFIX:
            raise TypeError(f"unsupported KV element type {dtype}")
        self.n_tokens, self.q_heads, self.kv_heads, self.head_dim = n_tokens, q_heads, kv_heads, head_dim
        self.block_size, self.dtype, self.num_blocks = block_size, dtype, num_blocks
        L = _lib.lib()
        self._streams = None        # handles of the streams that torch's allocator knows to use the workspace; the caller's own is the caller's
        if workspace is None:
            workspace = torch.empty(max(int(getattr(L, workspace_bytes)(n_tokens, q_heads, kv_heads, head_dim)), 256), dtype=torch.uint8, device=device)
            self._streams = {torch.cuda.current_stream(workspace.device).cuda_stream}
        self.workspace = workspace
        self._staging = _Staging(int(L.pkv_segment_staging_bytes(n_tokens, q_heads, kv_heads)))
        self.staging = self._staging.bytes
        self.plan = _lib.SegmentPlan()
        self._plan_ref = C.byref(self.plan)
        self._device, self._ws = workspace.get_device(), (_ptr(workspace), workspace.numel())
        self._out_elems = n_tokens * q_heads * head_dim
        self._block_elems = block_size * kv_heads * head_dim

    def _geometry(self):
        return self.q_heads, self.kv_heads, self.head_dim, self.block_size, self.dtype.itemsize

    def _build(self, name, image: bool, *args, stream=None):
        self._staging.writable()
        where = (self.staging.data_ptr(), self.staging.numel())
        L = _lib.lib()
        if image:
            st = getattr(L, name + "_image")(*args, *where, self.workspace.numel(), C.byref(self.plan))
        else:
            device = self.workspace.get_device()
            with _this_device(device) or contextlib.nullcontext():
                st = getattr(L, name)(*args, *where, _ptr(self.workspace), self.workspace.numel(), _stream(stream), C.byref(self.plan))
                self._staging.sent(stream, device)
                self._used_on(stream, device)
        _lib.check(name, st)
        self.plan.num_blocks = self.num_blocks

    def _used_on(self, stream, device: int) -> None:
        """Dropped, the workspace is not handed out again before `stream` is done with it.  (Of a bare handle nobody knows how long its
        stream lives: there the plan has to outlive the calls.)"""
        handle = _stream_of(stream, device)
        if self._streams is not None and handle not in self._streams and (stream is None or hasattr(stream, "cuda_stream")):
            self._streams.add(handle)
            self.workspace.record_stream(_torch.cuda.current_stream(device) if stream is None else stream)

    def _run(self, op, q, k_cache, v_cache, out, ints, scale, stream):
        """One attention call: pointers of q, the pools, the index arrays and out, in the order of the C signatures."""
        device = self._device
        other = _this_device(device)
        if other is not None:
            with other:
                return self._run(op, q, k_cache, v_cache, out, ints, scale, stream)
        _check((q, k_cache, v_cache, out), self.dtype, device, "q, out and pools")
        _check(ints, _torch.int32, device, "index arrays")
        if q.numel() < self._out_elems or out.numel() < self._out_elems:
            raise ValueError(f"q and out must have {self.n_tokens} rows of {self.q_heads} heads")
        pool = k_cache.numel()
        if v_cache.numel() != pool:
            raise ValueError("K and V pools differ in size")
        if self.plan.num_blocks * self._block_elems > pool:
            raise ValueError(f"the pools are smaller than the plan's {self.plan.num_blocks} blocks")
        fn, call = _fn(op, k_cache)
        handle = _stream_of(stream, device)
        if self._streams is not None and handle not in self._streams:
            self._used_on(stream, device)
        st = call(self._plan_ref, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), *[t.data_ptr() for t in ints], out.data_ptr(), scale,
                  *self._ws, handle)
        if st:
            _lib.check(fn, st)


class CrossPlan(_SegmentPlan):
    """Attention of each sequence's rows to the states of another sequence (an encoder's output), whose K and V lie
    in blocks of the pools: no causal mask, lengths of their own.  n_tokens: rows of q and out."""

    def __init__(self, n_tokens: int, n_seqs: int, q_heads: int, kv_heads: int, head_dim: int, block_size: int, dtype, num_blocks: int = 0,
                 workspace=None, device="cuda"):
        super().__init__("pkv_cross_workspace_bytes", n_tokens, q_heads, kv_heads, head_dim, block_size, dtype, num_blocks, workspace, device)
        self.n_seqs = n_seqs

    def _lengths(self, q_len, kv_len, q_start):
        arrays = [None if a is None else _int32(a) for a in (q_start, q_len, kv_len)]
        for a in arrays:
            if a is not None and a.shape != (self.n_seqs,):
                raise ValueError(f"the plan is for {self.n_seqs} sequences")
        return arrays

    def build_host(self, q_len, kv_len, q_start=None, stream=None) -> "CrossPlan":
        """q_len, kv_len, q_start: per sequence, on the host; without q_start the rows are packed one sequence behind
        the other.  Waits, if need be, until the plan's last upload has run."""
        arrays = self._lengths(q_len, kv_len, q_start)
        self._build("pkv_cross_plan_host", False, *[None if a is None else a.ctypes.data for a in arrays], self.n_seqs, self.n_tokens,
                    *self._geometry(), stream=stream)
        return self

    def build_host_image(self, q_len, kv_len, q_start=None) -> int:
        """The plan without the upload: bytes of self.staging that must reach the start of self.workspace, before the plan
        is made anew."""
        arrays = self._lengths(q_len, kv_len, q_start)
        self._build("pkv_cross_plan_host", True, *[None if a is None else a.ctypes.data for a in arrays], self.n_seqs, self.n_tokens,
                    *self._geometry())
        return int(self.plan.image_bytes)

    def attention(self, q, k_cache, v_cache, block_tables, table_offset, out, scale: float, stream=None) -> None:
        """out[t] = softmax(q[t] K^T scale) V over all keys of t's sequence; zero where it has none.  table_offset[s] is the
        start of sequence s's table."""
        if table_offset.numel() < self.n_seqs:
            raise ValueError(f"table_offset must name the tables of {self.n_seqs} sequences")
        self._run("pkv_cross_attn_", q, k_cache, v_cache, out, (block_tables, table_offset), scale, stream)


class PrefixPlan(_SegmentPlan):
    """Decode attention of tokens whose sequences all begin with the same blocks.  16-bit K/V at head_dim 64 or 128 in blocks of a power
    of two of at least 16 slots: the prefix is worked through once for all of them, where that is reckoned to pay; else
    as launch_attention_decode.  A captured call serves the step it was captured in."""

    def __init__(self, n_tokens: int, q_heads: int, kv_heads: int, head_dim: int, block_size: int, dtype, num_blocks: int = 0, workspace=None,
                 device="cuda"):
        super().__init__("pkv_prefix_workspace_bytes", n_tokens, q_heads, kv_heads, head_dim, block_size, dtype, num_blocks, workspace, device)

    def _positions(self, token_pos):
        pos = _int32(token_pos)
        if pos.shape != (self.n_tokens,):
            raise ValueError(f"the plan is for {self.n_tokens} tokens")
        return pos

    def build_host(self, token_pos, prefix_len: int, stream=None) -> "PrefixPlan":
        """token_pos: every token's position, on the host; its sequence's first prefix_len positions lie in the same
        blocks as everyone's.  Waits, if need be, until the plan's last upload has run."""
        pos = self._positions(token_pos)
        self._build("pkv_prefix_plan_host", False, pos.ctypes.data, self.n_tokens, prefix_len, *self._geometry(), stream=stream)
        return self

    def build_host_image(self, token_pos, prefix_len: int) -> int:
        """The plan without the upload: bytes of self.staging that must reach the start of self.workspace, before the plan
        is made anew."""
        pos = self._positions(token_pos)
        self._build("pkv_prefix_plan_host", True, pos.ctypes.data, self.n_tokens, prefix_len, *self._geometry())
        return int(self.plan.image_bytes)

    def attention(self, q, k_cache, v_cache, block_tables, table_offset, token_seq, out, scale: float, stream=None) -> None:
        """As launch_attention_decode with the step's whole tables."""
        if token_seq.numel() < self.n_tokens:
            raise ValueError(f"token_seq must name the sequences of {self.n_tokens} tokens")
        self._run("pkv_prefix_attn_", q, k_cache, v_cache, out, (block_tables, table_offset, token_seq), scale, stream)


def launch_attention_prefill(q, k_cache, v_cache, block_tables, table_offset, q_start, q_len, ctx_len, out,
                             n_tokens: int, n_seqs: int, max_q_len: int, q_heads: int, kv_heads: int, head_dim: int,
                             block_size: int, num_blocks: int, scale: float, stream=None) -> None:
    """Causal attention of each sequence's new chunk over its cached plus new tokens."""
    fn, call = _fn("pkv_prefill_attn_", k_cache)
    st = call(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables), _ptr(table_offset),
              _ptr(q_start), _ptr(q_len), _ptr(ctx_len), _ptr(out), n_tokens, n_seqs, max_q_len, q_heads,
              kv_heads, head_dim, block_size, num_blocks, C.c_float(scale), _stream(stream))
    _lib.check(fn, st)


def launch_copy_blocks(k_cache, v_cache, src_dst_pairs, n_pairs: int, block_size: int, kv_dim: int,
                       stream=None) -> None:
    """Copy-on-write: block pairs[2i] -> block pairs[2i+1] in both pools."""
    fn, call = _fn("pkv_copy_blocks_", k_cache)
    st = call(_ptr(k_cache), _ptr(v_cache), _ptr(src_dst_pairs), n_pairs, block_size, kv_dim,
              _stream(stream))
    _lib.check(fn, st)


def launch_copy_blocks_layers(cache_ptrs, n_caches: int, src_dst_pairs, n_pairs: int, block_bytes: int,
                              stream=None) -> None:
    """Same for every pool at once; cache_ptrs is an int64 CUDA tensor of pool base addresses."""
    st = _lib.lib().pkv_copy_blocks_layers(_ptr(cache_ptrs), n_caches, _ptr(src_dst_pairs), n_pairs, block_bytes,
                                           _stream(stream))
    _lib.check("pkv_copy_blocks_layers", st)


def debug_device_flags() -> int:
    """Reads and clears the word in which kernels record a bounded wait that ran out
    (synchronises the device; 0 = no kernel ever gave up)."""
    v = C.c_uint(0)
    _lib.check("pkv_debug_device_flags", _lib.lib().pkv_debug_device_flags(C.byref(v)))
    return int(v.value)
