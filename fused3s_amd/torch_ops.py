"""PyTorch-ROCm binding of the fused pass, for a graph-transformer layer.

The reference has no framework binding; its natural caller is a graph
attention layer: a QKV projection GEMM, the fused sparse attention over the
graph's edges, and an output projection.  Here torch supplies the device
memory and the stream; the attention is the HIP library's planned pass
(f3s_attention_fwd_planned), called on torch's current stream with the
tensors' device pointers, and the layer's projections are its f3s_linear_f16
(torch.nn.Linear's own product where that kernel is not the better one).  There
is no CPU fallback, and that pass is forward-only: calling it on tensors that require grad raises.
Differential attention (two softmax maps per head and their difference), edge
attention (one map, scores capped and lowered by distance), linear(), a projection
with bias, activation and residual, layer_norm() and linear_cross_entropy(), a
classifier's loss without its logits, have gradients.

    graph = TorchGraph(row_ptr, col_idx, heads=4)      # convert + plan + compile once
    o = graph.attention(q, k, v)                       # q/k/v [n, H, 64] fp16 -> fp32
    layer = GraphTransformerLayer(in_dim, heads=4).cuda().half()
    y = layer(x, graph)                                # x [n, in_dim] fp16

    o = graph.diff_attention(q, k, v, lam)             # q/k/v [n, H, 128] fp16 or bf16, autograd
    y = linear(x, weight, bias, "gelu", residual)      # autograd
    layer = DiffGraphTransformerLayer(in_dim, heads=4, ffn_dim=512).cuda().bfloat16()

    o = graph.edge_attention(q, k, v, 0.125, cap=30.0, positions=t, slopes=s)   # [n, H, 64]
    y = layer_norm(x, weight, bias)                    # float16, bfloat16 or float32
    loss = linear_cross_entropy(x, weight, classes)    # mean of the rows' losses
    layer = EdgeGraphTransformerLayer(in_dim, heads=4, ffn_dim=512, distance=True)

The drop-in launch is also a registered torch operator, on the block-sparse
form held in torch tensors (no plan, no state between calls):

    offs, bcol, mask = to_block_sparse(row_ptr, col_idx)        # GPU converter
    o = torch.ops.fused3s.attention_fwd(q, k, v, offs, bcol, mask, order, scale)
"""
from __future__ import annotations

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.fx import _symbolic_trace
from torch.utils._device import DeviceContext

# torch ships its own HIP runtime (torch/lib/libamdhip64.so, soname
# libamdhip64.so.7).  libf3s_hip.so binds to whichever libamdhip64.so.7 the
# process loaded first, so torch must be imported before the library's first
# GPU call; loaded the other way round, the process holds two HIP runtimes
# and torch sees no device.  Refuse that state with a clear message.


def _hip_runtimes() -> set[str]:
    try:
        with open("/proc/self/maps") as f:
            return {line.split()[-1] for line in f if "libamdhip64" in line}
    except OSError:
        return set()


if len(_hip_runtimes()) > 1:
    raise ImportError("two HIP runtimes are loaded (" + ", ".join(sorted(_hip_runtimes())) +
                      "): import torch before the first fused3s_amd GPU call")

import contextlib
import ctypes as C
import functools

from . import _lib
from .attention import Plan
from .device import DeviceArray, Stream, check
from .graph import (DeviceBSF, DeviceCSR, convert_device, converts_once, lists_oversized,
                    most_tiles, window_order_device)

HEAD_DIM = 64

# torch's current stream on a device as a number, without a Stream object around it
# (a small graph's pass is shorter than making one)
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


_NO_CONTEXT = contextlib.nullcontext()

_dispatch_modes, _is_tracing = torch._C._len_torch_dispatch_stack, torch._C._is_tracing
_transform, _dynamo = torch._C._functorch.peek_interpreter_stack, torch.compiler.is_dynamo_compiling


def _records_or_replaces() -> bool:
    """Whether a dispatch mode that records a program or stands in for its memory
    is active (make_fx, export, fake tensors; one that only looks on is neither)."""
    key = torch._C._TorchDispatchModeKey
    return any(torch._C._get_dispatch_mode(k) is not None
               for k in (key.PROXY, key.FAKE, key.FUNCTIONAL))


def _transformed(tensors) -> bool:
    f = torch._C._functorch
    return (any(t is not None and f.is_functorch_wrapped_tensor(t) for t in tensors)
            or any(i.key() == f.TransformType.Functionalize for i in f.get_interpreter_stack()))


_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter, type(None)))


def _stands_for_others(t: torch.Tensor) -> bool:
    """Whether t is of a subclass that dispatches its operations itself: its own
    data pointer is not what it stands for."""
    return type(t).__torch_dispatch__ is not torch.Tensor.__torch_dispatch__


def _refuse_unseen(who: str, *tensors) -> None:
    """Raises where torch does not see what a kernel called on data pointers does,
    and would go on without it: a forward-mode derivative would be lost, a traced
    program hold the output's allocation and nothing that fills it, a wrapper's
    tensor be left out.  (Some 0.7 us.)"""
    compiled = _dynamo()   # (it sees the level, not the tangents)
    if forward_ad._current_level >= 0 and (compiled or any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)):
        raise RuntimeError(f"{who} has no forward-mode derivative")
    if compiled:
        return   # (its graph breaks at the library's call, which then runs, or it raises)
    if (_is_tracing() or _symbolic_trace._is_fx_tracing_flag
            or _dispatch_modes() > 0 and _records_or_replaces()
            or _transform() is not None and _transformed(tensors)):
        raise RuntimeError(f"{who} cannot be traced or transformed: its kernel is not an operator "
                           "that torch sees")
    for t in tensors:
        if type(t) not in _PLAIN and _stands_for_others(t):
            raise TypeError(f"{who} takes no {type(t).__name__}: it has no memory of its own")


def _on(device: int):
    """The device as the current one (an autograd thread's own is that already)."""
    return _NO_CONTEXT if _current_device() == device else torch.cuda.device(device)


class _TorchStream(Stream):
    """torch's current HIP stream, viewed as a library Stream (not owned)."""

    def __init__(self, handle: int):   # noqa: D107 -- no stream is created
        self.handle = handle

    def __del__(self):
        pass


def current_stream() -> Stream:
    return _TorchStream(torch.cuda.current_stream().cuda_stream)


def _on_device(t, s: Stream) -> DeviceArray:
    """An int32 copy of an index array in library memory: from host memory, or
    device to device when it is a tensor of an index type on the current device
    already."""
    if torch.is_tensor(t):
        if (t.is_cuda and t.device.index == torch.cuda.current_device()
                and t.dtype in (torch.int32, torch.int64)):
            t = t.to(torch.int32).contiguous()
            a = DeviceArray(tuple(t.shape), np.int32)
            if a.nbytes:
                check(_lib.hip().f3s_memcpy_d2d(a.ptr, t.data_ptr(), a.nbytes, s.handle),
                      "f3s_memcpy_d2d")
            return a
        t = t.cpu().numpy()
    return DeviceArray.from_numpy(np.ascontiguousarray(t, np.int32), s)


def _device_csr(row_ptr, col_idx, s: Stream) -> DeviceCSR:
    csr = DeviceCSR.__new__(DeviceCSR)
    csr.row_ptr, csr.col_idx = _on_device(row_ptr, s), _on_device(col_idx, s)
    csr.n = csr.row_ptr.shape[0] - 1
    csr.nnz = csr.col_idx.shape[0]
    return csr


class TorchGraph:
    """A graph prepared once for repeated fused passes: CSR on the device,
    block-sparse form with row masks (GPU converter), descending-workload
    window order, and a compiled plan for `heads` heads of 64 dims.  A small
    graph's block-sparse lists keep the memory of a tile per edge (19 MB at most)."""

    def __init__(self, row_ptr, col_idx, heads: int = 1, masked: bool = True):
        if not torch.cuda.is_available():
            raise RuntimeError("TorchGraph needs a ROCm device (no CPU fallback)")
        s = current_stream()
        self.csr = _device_csr(row_ptr, col_idx, s)
        self.n = self.csr.n
        self.nnz = self.csr.nnz
        self.heads = heads
        self.masked = masked
        self.bsf: DeviceBSF = convert_device(self.csr, masks=True, stream=s)
        self.order = window_order_device(self.bsf, s)
        self.plan = Plan(self.bsf, self.order, H=heads, stream=s)
        if masked:
            self.plan.compile(s)
        self.device = torch.cuda.current_device()
        self._torch_device = torch.device("cuda", self.device)
        self._scheduled: Plan | None = None  # diff_attention's plan, where it is not self.plan
        self._reversed: Plan | None = None   # the reversed edges' (prepare_backward)
        self._workspace = {}
        self._edge_workspaces = {}

    def attention(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                  scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
        """softmax over each node's neighbours of scale * q.k, weights applied
        to v; [n, H, 64] fp16 contiguous CUDA tensors in, [n, H, 64] fp32 out.
        masked=False gives the reference's tile-dense semantics instead."""
        _refuse_unseen("attention", q, k, v)
        n, H = self.n, self.heads
        shape = (n, H, HEAD_DIM)
        for name, t in (("q", q), ("k", k), ("v", v)):
            if t.requires_grad:
                raise RuntimeError("the fused pass is forward-only (no autograd)")
            if t.dtype is not torch.float16 or not t.is_cuda or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous float16 CUDA tensor")
            if t.shape != shape and t.shape != (n, H * HEAD_DIM):   # (a Size is a tuple)
                raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
        if out is None:
            out = torch.empty(shape, dtype=torch.float32, device=q.device)
        elif (out.dtype != torch.float32 or not out.is_contiguous()
              or out.numel() != n * H * HEAD_DIM):
            raise ValueError("out must be a contiguous float32 tensor of n * H * 64 elements")
        # Plan.forward without its wrappers: a small graph's pass is shorter
        # than the Python around it
        bsf = self.bsf
        check(_lib.hip().f3s_attention_fwd_planned(
            self.plan.handle, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            bsf.block_col.ptr, bsf.tile_mask.ptr if self.masked else None, n, HEAD_DIM, H, scale,
            _raw_stream(_current_device())), "f3s_attention_fwd_planned")
        return out

    def takes_packed(self) -> bool:
        """Whether attention_packed takes this graph: masked semantics, and
        the packed tensor within the 32-bit offsets of its launch."""
        return self.masked and 3 * self.n * self.heads * 2 * HEAD_DIM <= 0xffff4000

    def attention_packed(self, qkv: torch.Tensor, scale: float = 1.0,
                         dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """attention() on the [n, 3 * H * 64] fp16 output of one projection
        (q, k and v side by side in each row, no copies made), O [n, H, 64]
        in float32 or float16 (f3s_attention_fwd_packed)."""
        _refuse_unseen("attention_packed", qkv)
        if qkv.requires_grad:
            raise RuntimeError("the fused pass is forward-only (no autograd)")
        if qkv.dtype != torch.float16 or not qkv.is_cuda or not qkv.is_contiguous():
            raise ValueError("qkv must be a contiguous float16 CUDA tensor")
        if tuple(qkv.shape) != (self.n, 3 * self.heads * HEAD_DIM):
            raise ValueError(f"qkv must have shape {(self.n, 3 * self.heads * HEAD_DIM)}, "
                             f"got {tuple(qkv.shape)}")
        if dtype not in (torch.float32, torch.float16):
            raise ValueError("dtype must be float32 or float16")
        out = torch.empty((self.n, self.heads, HEAD_DIM), dtype=dtype, device=qkv.device)
        if self.n:
            check(_lib.hip().f3s_attention_fwd_packed(
                self.plan.handle, qkv.data_ptr(), out.data_ptr(), int(dtype == torch.float16),
                self.n, HEAD_DIM, self.heads, float(scale),
                _raw_stream(_current_device())), "f3s_attention_fwd_packed")
        return out

    def prepare_backward(self) -> "TorchGraph":
        """Builds what the gradients of diff_attention and edge_attention read, a
        compiled plan of the reversed edges; the first call that needs it does so otherwise.
        Waits for the GPU, so before a capture.  (The leaves of a captured step
        must not belong to an eager step that is still alive, as with torch's
        own operators: capture with detached ones.  A captured call reads this
        object's lists, so it has to outlive the replays.)"""
        if self._reversed is None:
            if not self.masked:
                raise ValueError("a gradient needs the masked (edge-exact) semantics")
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("call prepare_backward() before the capture")
            with torch.cuda.device(self.device):
                s = current_stream()
                csr, rev = self.csr, DeviceCSR.__new__(DeviceCSR)
                rev.n, rev.nnz = csr.n, csr.nnz
                rev.row_ptr = DeviceArray(csr.n + 1, np.int32)
                rev.col_idx = DeviceArray(csr.nnz, np.int32)
                check(_lib.hip().f3s_reverse_csr(csr.row_ptr.ptr, csr.col_idx.ptr, csr.n, csr.nnz,
                                                 rev.row_ptr.ptr, rev.col_idx.ptr, s.handle),
                      "f3s_reverse_csr")
                bsf = convert_device(rev, masks=True, stream=s)
                self._diff_plan()
                self._reversed = self._compiled(bsf, s)
        return self

    def _compiled(self, bsf: DeviceBSF, s: Stream) -> Plan:
        """A compiled plan in the library's sequence (in natural order up to 512
        windows), its windows cut finer; small graphs' teams are the same in every
        sequence."""
        plan = Plan(bsf, H=self.heads, stream=s, scheduled=True)
        plan.compile(s)
        plan.bsf = None   # the compiled lists are all that is read
        return plan

    def _diff_plan(self) -> Plan:
        """The plan of diff_attention and edge_attention: self.plan, where that follows the
        library's sequence or the windows run on teams; else one made for it by the
        first call (_compiled).  (Waits for the GPU then, so before a capture.)"""
        if self._scheduled is None:
            W = self.bsf.W
            if W * self.heads <= 1024 or W * self.heads >= 2**18:
                self._scheduled = self.plan
            else:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("call the operator once, or prepare_backward(), before "
                                       "the capture")
                self._scheduled = self._compiled(self.bsf, current_stream())
        return self._scheduled

    def _diff_workspace(self, backward: bool) -> torch.Tensor:
        size = self._workspace.get(backward)
        if size is None:
            need = C.c_int64()
            check(_lib.hip().f3s_diff_attention_workspace(
                self._diff_plan().handle, self._reversed.handle if backward else None,
                C.byref(need)),
                "f3s_diff_attention_workspace")
            size = self._workspace[backward] = need.value
        return torch.empty(size, dtype=torch.uint8, device=self._torch_device) if size else None

    def _check_exact(self, who: str) -> None:
        if not self.masked:
            raise ValueError(f"{who} is edge-exact: it needs masked=True")
        if _current_device() != self.device:
            raise ValueError(f"the graph is on device {self.device}, which is not the current one")

    def _check_diff(self, lam, tensors) -> None:
        """Raises for tensors (by name) that diff_attention does not take."""
        self._check_exact("differential attention")
        device = self._torch_device
        if lam.dtype is not torch.float32 or lam.device != device or lam.shape != (self.heads,):
            raise ValueError(f"lam must be a float32 tensor of {self.heads} weights on the graph's "
                             "device")
        self._check_halves(tensors)

    def _check_halves(self, tensors) -> None:
        device, dtype = self._torch_device, None
        for name, t, *shapes in tensors:
            if t.dtype not in _DTYPES or t.device != device or (dtype or t.dtype) is not t.dtype:
                raise ValueError(f"{name} must be a float16 or bfloat16 tensor on the graph's "
                                 "device, all of one type")
            dtype = t.dtype
            if t.shape not in shapes:
                raise ValueError(f"{name} must have shape {shapes[0]}, got {tuple(t.shape)}")

    def diff_attention(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor,
                       scale: float = 1.0) -> torch.Tensor:
        """Differential attention over each node's neighbours: per head two maps
        of 64 dims, the halves of q and k, and values of 128,
        (softmax(scale * q1.k1) - lam[h] * softmax(scale * q2.k2)) v.
        q, k, v: float16 or bfloat16 CUDA tensors [n, H, 128], each row's heads
        contiguous, rows at any distance of a multiple of 8 values (a slice of a
        projection's output is taken as it is; other layouts are copied);
        lam: float32 [H].  Returns [n, H, 128] in q's type: sums in float32,
        rounded once; nodes without edges get 0.  (Logits are float32: past 2^24 in
        size the weights are not resolved.)  Differentiable in q, k, v and
        lam (once); tracing, functorch's transforms and forward-mode differentiation
        are refused.  A graph serves any number of calls at once."""
        _refuse_unseen("diff_attention", q, k, v, lam)
        shape, flat = (self.n, self.heads, 2 * HEAD_DIM), (self.n, self.heads * 2 * HEAD_DIM)
        self._check_diff(lam, (("q", q, shape, flat), ("k", k, shape, flat), ("v", v, shape, flat)))
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                        or lam.requires_grad):
            self.prepare_backward()
            return _DiffAttention.apply(self, float(scale), lam, q, k, v)
        return _diff_forward(self, float(scale), lam, *(_rows(t, self) for t in (q, k, v)))

    def diff_attention_packed(self, qkv: torch.Tensor, lam: torch.Tensor,
                              scale: float = 1.0) -> torch.Tensor:
        """diff_attention() on the [n, 3 * H * 128] output of one projection (q,
        k and v side by side in each row), whose gradient is then one tensor
        too, written in place of its thirds."""
        _refuse_unseen("diff_attention_packed", qkv, lam)
        self._check_diff(lam, (("qkv", qkv, (self.n, 3 * self.heads * 2 * HEAD_DIM)),))
        if torch.is_grad_enabled() and (qkv.requires_grad or lam.requires_grad):
            self.prepare_backward()
            return _DiffAttention.apply(self, float(scale), lam, qkv)
        return _diff_forward(self, float(scale), lam, *_thirds(qkv, self))

    def _check_edge(self, cap, positions, slopes, tensors):
        """Raises for what edge_attention does not take (tensors by name); its bias as
        (cap, dims, positions, slopes)."""
        self._check_exact("edge attention")
        self._check_halves(tensors)
        cap = 0.0 if cap is None else float(cap)
        if not (cap == 0.0 or 1e-30 < cap < 1e30):
            raise ValueError(f"cap must be positive (None or 0: none), got {cap}")
        if (positions is None) != (slopes is None):
            raise ValueError("positions and slopes come together")
        if positions is None:
            return cap, 0, None, None
        device = self._torch_device
        if (positions.dtype is not torch.float32 or positions.device != device
                or positions.dim() not in (1, 2) or positions.shape[0] != self.n
                or positions.dim() == 2 and not 1 <= positions.shape[1] <= 3):
            raise ValueError(f"positions must be a float32 tensor of {self.n} nodes' 1 to 3 "
                             "coordinates on the graph's device")
        if positions.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("edge attention has no gradient of positions: detach them")
        if (slopes.dtype is not torch.float32 or slopes.device != device
                or slopes.shape != (self.heads,)):
            raise ValueError(f"slopes must be a float32 tensor of {self.heads} weights on the "
                             "graph's device")
        return (cap, 1 if positions.dim() == 1 else positions.shape[1], positions.contiguous(),
                slopes)

    def edge_attention(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float = 1.0,
                       cap: float | None = None, positions: torch.Tensor | None = None,
                       slopes: torch.Tensor | None = None) -> torch.Tensor:
        """Softmax attention over each node's neighbours j, trainable: the weights of v
        are the softmax of
            cap * tanh(scale * q.k / cap) - slopes[h] * |positions[i] - positions[j]|
        (cap None: scale * q.k itself; positions None: no distances).
        q, k, v: float16 or bfloat16 CUDA tensors [n, H, 64], each row's heads
        contiguous, rows at any distance of a multiple of 8 values (a slice of a
        projection's output is taken as it is; other layouts are copied); positions:
        float32 [n] (times, say) or [n, 1 to 3] (points); slopes: float32 [H].  Where
        slopes are positive, a node with an infinite coordinate is taken out of the graph.
        Returns [n, H, 64] in q's type: sums in float32, rounded once; nodes without
        edges get 0.  Differentiable in q, k, v and slopes (once); tracing, functorch's
        transforms and forward-mode differentiation are refused.  A graph serves any
        number of calls at once."""
        _refuse_unseen("edge_attention", q, k, v, positions, slopes)
        shape, flat = (self.n, self.heads, HEAD_DIM), (self.n, self.heads * HEAD_DIM)
        bias = self._check_edge(cap, positions, slopes,
                                (("q", q, shape, flat), ("k", k, shape, flat), ("v", v, shape, flat)))
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                        or slopes is not None and slopes.requires_grad):
            self.prepare_backward()
            return _EdgeAttention.apply(self, float(scale), *bias, q, k, v)
        return _edge_forward(self, float(scale), *bias, *(_rows(t, self, HEAD_DIM)
                                                          for t in (q, k, v)))

    def edge_attention_packed(self, qkv: torch.Tensor, scale: float = 1.0,
                              cap: float | None = None, positions: torch.Tensor | None = None,
                              slopes: torch.Tensor | None = None) -> torch.Tensor:
        """edge_attention() on the [n, 3 * H * 64] output of one projection (q, k and v
        side by side in each row), whose gradient is then one tensor too, written in
        place of its thirds."""
        _refuse_unseen("edge_attention_packed", qkv, positions, slopes)
        bias = self._check_edge(cap, positions, slopes,
                                (("qkv", qkv, (self.n, 3 * self.heads * HEAD_DIM)),))
        if torch.is_grad_enabled() and (qkv.requires_grad
                                        or slopes is not None and slopes.requires_grad):
            self.prepare_backward()
            return _EdgeAttention.apply(self, float(scale), *bias, qkv)
        return _edge_forward(self, float(scale), *bias, *_thirds(qkv, self, HEAD_DIM))

    def _edge_workspace(self, backward: bool, dims: int) -> torch.Tensor:
        size = self._edge_workspaces.get((backward, dims))
        if size is None:
            need = C.c_int64()
            check(_lib.hip().f3s_edge_attention_workspace(
                self._diff_plan().handle, self._reversed.handle if backward else None, dims,
                C.byref(need)),
                "f3s_edge_attention_workspace")
            size = self._edge_workspaces[backward, dims] = need.value
        return torch.empty(size, dtype=torch.uint8, device=self._torch_device) if size else None


_DTYPES = {torch.float16: 0, torch.bfloat16: 1}   # F3S_F16, F3S_BF16


def _rows(t: torch.Tensor, graph: TorchGraph, per_head: int = 2 * HEAD_DIM) -> torch.Tensor:
    """[n, width] with each row contiguous, 16-byte aligned: t itself where its
    layout is that already."""
    n, width = graph.n, graph.heads * per_head
    if t.is_contiguous() and t.stride(0) == width and t.data_ptr() % 16 == 0:
        return t.view(n, width) if t.dim() == 3 else t
    if t.dim() == 3 and (t.stride(2) != 1 or t.stride(1) != per_head and graph.heads > 1):
        t = t.contiguous()
    if t.dim() == 3:
        t = t.as_strided((n, width), (t.stride(0), 1))
    if t.stride(1) != 1 or t.data_ptr() % 16 or n > 1 and (t.stride(0) % 8
                                                           or t.stride(0) < width):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _thirds(qkv: torch.Tensor, graph: TorchGraph, per_head: int = 2 * HEAD_DIM):
    width = graph.heads * per_head
    if qkv.stride(-1) != 1 or qkv.data_ptr() % 16 or (
            graph.n > 1 and (qkv.stride(0) % 8 or qkv.stride(0) < 3 * width)):
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    return tuple(qkv[:, i * width:(i + 1) * width] for i in range(3))


def _stride(t: torch.Tensor, n: int) -> int:
    """Values between the n rows (a single row's stride is of any size and not used)."""
    return t.stride(0) if n > 1 else t.shape[1]


def _diff_forward(graph: TorchGraph, scale: float, lam, q, k, v, lse=None) -> torch.Tensor:
    n, H = graph.n, graph.heads
    out = q.new_empty((n, H, 2 * HEAD_DIM))
    if n:
        plan = graph._diff_plan().handle
        ws = graph._diff_workspace(False)
        if not lam.is_contiguous():
            lam = lam.contiguous()
        check(_lib.hip().f3s_diff_attention_fwd(
            plan, q.data_ptr(), _stride(q, n), k.data_ptr(), _stride(k, n), v.data_ptr(),
            _stride(v, n), lam.data_ptr(), out.data_ptr(), H * 2 * HEAD_DIM,
            None if lse is None else lse.data_ptr(), _DTYPES[q.dtype], n, H, scale,
            None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(),
            _raw_stream(graph.device)), "f3s_diff_attention_fwd")
    return out


class _DiffAttention(torch.autograd.Function):
    """diff_attention and its gradient; one packed tensor or three."""

    @staticmethod
    def forward(ctx, graph, scale, lam, *tensors):
        packed = len(tensors) == 1
        rows = _thirds(tensors[0], graph) if packed else [_rows(t, graph) for t in tensors]
        lse = torch.empty((graph.n, graph.heads, 2), dtype=torch.float32, device=lam.device)
        lam = lam.contiguous()
        out = _diff_forward(graph, scale, lam, *rows, lse=lse)
        ctx.graph, ctx.scale, ctx.shapes = graph, scale, [t.shape for t in tensors]
        ctx.save_for_backward(lam, lse, *tensors)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        graph, n, H = ctx.graph, ctx.graph.n, ctx.graph.heads
        width = H * 2 * HEAD_DIM
        lam, lse, *tensors = ctx.saved_tensors
        packed = len(tensors) == 1
        q, k, v = _thirds(tensors[0], graph) if packed else (_rows(t, graph) for t in tensors)
        grads = [q.new_empty(shape) for shape in ctx.shapes]
        if packed:
            dq, dk, dv = (grads[0][:, i * width:(i + 1) * width] for i in range(3))
        else:
            dq, dk, dv = (t.view(n, width) for t in grads)
        dlam = torch.empty_like(lam)
        do = _rows(grad, graph)
        with _on(graph.device):
            ws = graph._diff_workspace(True)
            check(_lib.hip().f3s_diff_attention_bwd(
                graph._diff_plan().handle, graph._reversed.handle, q.data_ptr(), _stride(q, n),
                k.data_ptr(), _stride(k, n), v.data_ptr(), _stride(v, n), lam.data_ptr(),
                lse.data_ptr(), do.data_ptr(), _stride(do, n), dq.data_ptr(), _stride(dq, n),
                dk.data_ptr(), _stride(dk, n), dv.data_ptr(), _stride(dv, n), dlam.data_ptr(),
                _DTYPES[q.dtype], n, H, ctx.scale,
                ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
                _raw_stream(graph.device)), "f3s_diff_attention_bwd")
        return None, None, dlam, *grads


def _edge_forward(graph: TorchGraph, scale: float, cap, dims, positions, slopes, q, k, v,
                  lse=None) -> torch.Tensor:
    n, H = graph.n, graph.heads
    out = q.new_empty((n, H, HEAD_DIM))
    if n:
        plan = graph._diff_plan().handle
        ws = graph._edge_workspace(False, dims)
        if dims and not slopes.is_contiguous():
            slopes = slopes.contiguous()
        check(_lib.hip().f3s_edge_attention_fwd(
            plan, q.data_ptr(), _stride(q, n), k.data_ptr(), _stride(k, n), v.data_ptr(),
            _stride(v, n), out.data_ptr(), H * HEAD_DIM, None if lse is None else lse.data_ptr(),
            _DTYPES[q.dtype], n, H, scale, cap, positions.data_ptr() if dims else None, dims,
            slopes.data_ptr() if dims else None, None if ws is None else ws.data_ptr(),
            0 if ws is None else ws.numel(), _raw_stream(graph.device)), "f3s_edge_attention_fwd")
    return out


class _EdgeAttention(torch.autograd.Function):
    """edge_attention and its gradient; one packed tensor or three."""

    @staticmethod
    def forward(ctx, graph, scale, cap, dims, positions, slopes, *tensors):
        rows = (_thirds(tensors[0], graph, HEAD_DIM) if len(tensors) == 1
                else [_rows(t, graph, HEAD_DIM) for t in tensors])
        lse = torch.empty((graph.n, graph.heads), dtype=torch.float32, device=tensors[0].device)
        if dims:
            slopes = slopes.contiguous()
        out = _edge_forward(graph, scale, cap, dims, positions, slopes, *rows, lse=lse)
        ctx.graph, ctx.scale, ctx.cap, ctx.dims = graph, scale, cap, dims
        ctx.shapes = [t.shape for t in tensors]
        ctx.save_for_backward(positions, slopes, lse, *tensors)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        graph, n, H, dims = ctx.graph, ctx.graph.n, ctx.graph.heads, ctx.dims
        width = H * HEAD_DIM
        positions, slopes, lse, *tensors = ctx.saved_tensors
        packed = len(tensors) == 1
        q, k, v = (_thirds(tensors[0], graph, HEAD_DIM) if packed
                   else (_rows(t, graph, HEAD_DIM) for t in tensors))
        grads = [q.new_empty(shape) for shape in ctx.shapes]
        if packed:
            dq, dk, dv = (grads[0][:, i * width:(i + 1) * width] for i in range(3))
        else:
            dq, dk, dv = (t.view(n, width) for t in grads)
        dslopes = torch.empty_like(slopes) if dims else None
        do = _rows(grad, graph, HEAD_DIM)
        with _on(graph.device):
            ws = graph._edge_workspace(True, dims)
            check(_lib.hip().f3s_edge_attention_bwd(
                graph._diff_plan().handle, graph._reversed.handle, q.data_ptr(), _stride(q, n),
                k.data_ptr(), _stride(k, n), v.data_ptr(), _stride(v, n), lse.data_ptr(),
                do.data_ptr(), _stride(do, n), dq.data_ptr(), _stride(dq, n), dk.data_ptr(),
                _stride(dk, n), dv.data_ptr(), _stride(dv, n),
                dslopes.data_ptr() if dims else None, _DTYPES[q.dtype], n, H, ctx.scale, ctx.cap,
                positions.data_ptr() if dims else None, dims, slopes.data_ptr() if dims else None,
                ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
                _raw_stream(graph.device)), "f3s_edge_attention_bwd")
        return None, None, None, None, None, dslopes, *grads


# F3S_ACT_NONE ..
_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


@functools.lru_cache(maxsize=256)
def _linear_bytes(n, K, M, act, backward) -> int:
    need = C.c_int64()
    check(_lib.hip().f3s_linear_workspace(n, K, M, act, backward, C.byref(need)),
          "f3s_linear_workspace")
    return need.value


def _linear_workspace(n, K, M, act, backward, device):
    size = _linear_bytes(n, K, M, act, backward)
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _matrix(t: torch.Tensor) -> torch.Tensor:
    """A matrix whose rows are contiguous and do not overlap."""
    return t if t.stride(1) == 1 and (t.stride(0) >= t.shape[1] or t.shape[0] == 1) \
        else t.contiguous()


def _linear_forward(x, w, b, r, act):
    (n, K), M = x.shape, w.shape[0]
    y = x.new_empty((n, M))
    if n:
        ws = _linear_workspace(n, K, M, act, 0, x.device) if n > 64 else None
        check(_lib.hip().f3s_linear_fwd(
            x.data_ptr(), _stride(x, n), w.data_ptr(), b.data_ptr() if b is not None else None,
            r.data_ptr() if r is not None else None, _stride(r, n) if r is not None else 0,
            y.data_ptr(), n, K, M, act, _DTYPES[x.dtype],
            ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
            _raw_stream(x.device.index)), "f3s_linear_fwd")
    return y


class _Linear(torch.autograd.Function):
    """linear()'s matrices and their gradients."""

    @staticmethod
    def forward(ctx, x, w, b, r, act):
        ctx.act = act
        ctx.save_for_backward(x, w, b if act else None)
        return _linear_forward(x, w, b, r, act)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, w, b = ctx.saved_tensors
        (n, K), M, act = x.shape, w.shape[0], ctx.act
        needs = ctx.needs_input_grad
        empty = lambda wanted, *shape: x.new_empty(shape) if wanted else None
        dx, dw, db = empty(needs[0], n, K), empty(needs[1], M, K), empty(needs[2], M)
        if any(needs[:3]):
            dy = _matrix(grad)
            with _on(x.device.index):
                ws = _linear_workspace(n, K, M, act, 1, x.device)
                check(_lib.hip().f3s_linear_bwd(
                    x.data_ptr(), _stride(x, n), w.data_ptr(),
                    b.data_ptr() if b is not None else None, dy.data_ptr(), _stride(dy, n),
                    *(t.data_ptr() if t is not None else None for t in (dx, dw, db)), n, K, M, act,
                    _DTYPES[x.dtype], ws.data_ptr() if ws is not None else None,
                    ws.numel() if ws is not None else 0, _raw_stream(x.device.index)),
                    "f3s_linear_bwd")
        return dx, dw, db, grad if needs[3] else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           activation: str | None = None, residual: torch.Tensor | None = None) -> torch.Tensor:
    """activation(x @ weight.T + bias) + residual in one kernel: x [..., K],
    weight [M, K], bias [M], residual [..., M], all float16 or all bfloat16 on one
    GPU; activation None, "relu", "gelu", "gelu_tanh" or "silu".  Sums and
    epilogue are in float32, the result is rounded once.  Differentiable (once);
    for the backward pass the product z is computed again rather than kept, and
    dz = dy * activation'(z) is rounded to the type, as between torch's own
    modules, before the gradients of x and weight are made of it: those two are
    rounded twice, bias's gradient (and all of them without an activation) once.
    Tracing, functorch's transforms and forward-mode differentiation are refused."""
    _refuse_unseen("linear", x, weight, bias, residual)
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {list(_ACTIVATIONS)}, got {activation!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x [..., K] and weight [M, K] do not fit: {tuple(x.shape)}, "
                         f"{tuple(weight.shape)}")
    M, K = weight.shape
    if M == 0 or K == 0:
        raise ValueError("weight must not be empty")
    if bias is not None and bias.shape != (M,):
        raise ValueError(f"bias must have shape {(M,)}, got {tuple(bias.shape)}")
    flat = x.dim() == 2
    shape = (x.shape[0], M) if flat else (*x.shape[:-1], M)
    if residual is not None and residual.shape != shape:
        raise ValueError(f"residual must have shape {shape}, got {tuple(residual.shape)}")
    dtype, device = x.dtype, x.device
    if (dtype not in _DTYPES or not x.is_cuda
            or weight.dtype is not dtype or weight.device != device
            or bias is not None and (bias.dtype is not dtype or bias.device != device)
            or residual is not None and (residual.dtype is not dtype
                                         or residual.device != device)):
        raise ValueError("x, weight, bias and residual must be float16 or bfloat16 tensors on a "
                         "GPU, all of one type and on one device")
    if device.index != _current_device():
        with torch.cuda.device(device):
            return linear(x, weight, bias, activation, residual)
    x2 = _matrix(x if flat else x.reshape(-1, K))
    w = weight if weight.is_contiguous() else weight.contiguous()
    b = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    r = residual
    if r is not None:
        r = _matrix(r if flat else r.reshape(-1, M))
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or bias is not None and bias.requires_grad
                                    or residual is not None and residual.requires_grad):
        y = _Linear.apply(x2, w, b, r, act)
    else:
        y = _linear_forward(x2, w, b, r, act)
    return y if flat else y.view(shape)


_NORM_DTYPES = {**_DTYPES, torch.float32: 2}   # F3S_F32


@functools.lru_cache(maxsize=256)
def _norm_bytes(n, width, dtype) -> int:
    need = C.c_int64()
    check(_lib.hip().f3s_layer_norm_workspace(n, width, dtype, C.byref(need)),
          "f3s_layer_norm_workspace")
    return need.value


def _norm_forward(x, w, b, eps, stats=None):
    n, width = x.shape
    y = x.new_empty((n, width))
    if n:
        dtype = _NORM_DTYPES[x.dtype]
        of = w if w is not None else b
        check(_lib.hip().f3s_layer_norm_fwd(
            x.data_ptr(), _stride(x, n), w.data_ptr() if w is not None else None,
            b.data_ptr() if b is not None else None, y.data_ptr(),
            stats.data_ptr() if stats is not None else None, n, width, eps, dtype,
            dtype if of is None else _NORM_DTYPES[of.dtype], _raw_stream(x.device.index)),
            "f3s_layer_norm_fwd")
    return y


class _LayerNorm(torch.autograd.Function):
    """layer_norm()'s matrix and its gradients."""

    @staticmethod
    def forward(ctx, x, w, b, eps):
        stats = torch.empty((x.shape[0], 2), dtype=torch.float32, device=x.device)
        ctx.of = None if b is None else b.dtype
        ctx.save_for_backward(x, w, stats)
        return _norm_forward(x, w, b, eps, stats)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, w, stats = ctx.saved_tensors
        n, width = x.shape
        needs = ctx.needs_input_grad
        of = ctx.of if w is None else w.dtype
        dx = x.new_empty((n, width)) if needs[0] else None
        dw, db = (x.new_empty(width, dtype=of) if wanted else None for wanted in needs[1:3])
        if any(needs[:3]):
            dtype = _NORM_DTYPES[x.dtype]
            dy = _matrix(grad)
            with _on(x.device.index):
                ws = (torch.empty(_norm_bytes(n, width, dtype), dtype=torch.uint8, device=x.device)
                      if needs[1] or needs[2] else None)
                check(_lib.hip().f3s_layer_norm_bwd(
                    x.data_ptr(), _stride(x, n), w.data_ptr() if w is not None else None,
                    stats.data_ptr(), dy.data_ptr(), _stride(dy, n),
                    *(t.data_ptr() if t is not None else None for t in (dx, dw, db)), n, width,
                    dtype, dtype if of is None else _NORM_DTYPES[of],
                    ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
                    _raw_stream(x.device.index)), "f3s_layer_norm_bwd")
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension: x
    [..., width] float16, bfloat16 or float32 on a GPU, weight and bias [width], both of
    x's type or both float32.  Returns x's type; sums are float32, every result is
    rounded once.  Differentiable (once) in all three; the gradients of weight and
    bias are the same from run to run.  Tracing, functorch's transforms and
    forward-mode differentiation are refused."""
    _refuse_unseen("layer_norm", x, weight, bias)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must have a last dimension of at least 1, got {tuple(x.shape)}")
    width, dtype, device = x.shape[-1], x.dtype, x.device
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != (width,):
            raise ValueError(f"{name} must have shape {(width,)}, got {tuple(t.shape)}")
    of = weight if weight is not None else bias
    if (dtype not in _NORM_DTYPES or not x.is_cuda
            or of is not None and ((of.dtype is not dtype and of.dtype is not torch.float32)
                                   or of.device != device)
            or weight is not None and bias is not None and (bias.dtype is not weight.dtype
                                                            or bias.device != device)):
        raise ValueError("x must be a float16, bfloat16 or float32 tensor on a GPU, weight and bias "
                         "both of its type or both float32, on its device")
    if device.index != _current_device():
        with torch.cuda.device(device):
            return layer_norm(x, weight, bias, eps)
    x2 = _matrix(x if x.dim() == 2 else x.reshape(-1, width))
    w = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    b = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight is not None and weight.requires_grad
                                    or bias is not None and bias.requires_grad):
        y = _LayerNorm.apply(x2, w, b, float(eps))
    else:
        y = _norm_forward(x2, w, b, float(eps))
    return y if x.dim() == 2 else y.view(x.shape)


_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}   # F3S_LOSS_NONE ..


@functools.lru_cache(maxsize=256)
def _loss_bytes(n, K, V, backward) -> int:
    need = C.c_int64()
    check(_lib.hip().f3s_cross_entropy_workspace(n, K, V, backward, C.byref(need)),
          "f3s_cross_entropy_workspace")
    return need.value


def _loss_workspace(n, K, V, backward, device):
    size = _loss_bytes(n, K, V, backward)
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _loss_forward(x, w, b, target, ignore, reduction, lse=None):
    (n, K), V = x.shape, w.shape[0]
    loss = torch.empty(() if reduction else (n,), dtype=torch.float32, device=x.device)
    ws = _loss_workspace(n, K, V, 0, x.device)
    check(_lib.hip().f3s_cross_entropy_fwd(
        x.data_ptr(), _stride(x, n), w.data_ptr(), b.data_ptr() if b is not None else None,
        target.data_ptr(), ignore, loss.data_ptr(), lse.data_ptr() if lse is not None else None,
        n, K, V, reduction, _DTYPES[x.dtype], ws.data_ptr() if ws is not None else None,
        ws.numel() if ws is not None else 0, _raw_stream(x.device.index)), "f3s_cross_entropy_fwd")
    return loss


class _LinearCrossEntropy(torch.autograd.Function):
    """linear_cross_entropy()'s matrices and their gradients."""

    @staticmethod
    def forward(ctx, x, w, b, target, ignore, reduction):
        lse = torch.empty(x.shape[0] + 1, dtype=torch.float32, device=x.device)
        ctx.ignore, ctx.reduction = ignore, reduction
        ctx.save_for_backward(x, w, b, target, lse)
        return _loss_forward(x, w, b, target, ignore, reduction, lse)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, w, b, target, lse = ctx.saved_tensors
        (n, K), V = x.shape, w.shape[0]
        needs = ctx.needs_input_grad
        empty = lambda wanted, *shape: x.new_empty(shape) if wanted else None
        dx, dw, db = empty(needs[0], n, K), empty(needs[1], V, K), empty(needs[2], V)
        if any(needs[:3]):
            grad = grad.contiguous()
            with _on(x.device.index):
                ws = _loss_workspace(n, K, V, 1, x.device)
                check(_lib.hip().f3s_cross_entropy_bwd(
                    x.data_ptr(), _stride(x, n), w.data_ptr(),
                    b.data_ptr() if b is not None else None, target.data_ptr(), ctx.ignore,
                    lse.data_ptr(), grad.data_ptr(),
                    *(t.data_ptr() if t is not None else None for t in (dx, dw, db)), n, K, V,
                    ctx.reduction, _DTYPES[x.dtype], ws.data_ptr() if ws is not None else None,
                    ws.numel() if ws is not None else 0, _raw_stream(x.device.index)),
                    "f3s_cross_entropy_bwd")
        return dx, dw, db, None, None, None


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         bias: torch.Tensor | None = None, ignore_index: int = -100,
                         reduction: str = "mean") -> torch.Tensor:
    """The cross entropy of the logits x @ weight.T + bias with the classes `target`,
    without keeping the logits: x [..., K], weight [V, K], bias [V], all float16 or all
    bfloat16 on one GPU, target [...] int64.  Rows of ignore_index have no loss and no
    gradient; a target that is no class has NaN as both.  reduction "mean" (over the
    rows that are not ignored), "sum" or "none"; float32.  (An ignored row's x is
    multiplied by 0 in weight's gradient: infinite or NaN values of it are NaN there, as
    in torch.)  Logits are not rounded, sums are float32.  Differentiable (once) in x, weight and bias; for the backward pass the
    logits are computed again, some classes at a time, and their gradient (up to what
    multiplies all of it: the mean's divisor, a loss scale) is rounded to the type before
    the gradients of x and weight are made of it, so these two are rounded twice (once
    where V is 64 and K 256 at most, K a multiple of 8).
    Tracing, functorch's transforms and forward-mode differentiation are refused."""
    _refuse_unseen("linear_cross_entropy", x, weight, target, bias)
    how = _REDUCTIONS.get(reduction)
    if how is None:
        raise ValueError(f"reduction must be one of {list(_REDUCTIONS)}, got {reduction!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x [..., K] and weight [V, K] do not fit: {tuple(x.shape)}, "
                         f"{tuple(weight.shape)}")
    V, K = weight.shape
    if V == 0 or K == 0:
        raise ValueError("weight must not be empty")
    if bias is not None and bias.shape != (V,):
        raise ValueError(f"bias must have shape {(V,)}, got {tuple(bias.shape)}")
    if target.shape != x.shape[:-1]:
        raise ValueError(f"target must have shape {tuple(x.shape[:-1])}, got {tuple(target.shape)}")
    dtype, device = x.dtype, x.device
    if (dtype not in _DTYPES or not x.is_cuda
            or weight.dtype is not dtype or weight.device != device
            or bias is not None and (bias.dtype is not dtype or bias.device != device)):
        raise ValueError("x, weight and bias must be float16 or bfloat16 tensors on a GPU, all of "
                         "one type and on one device")
    if target.dtype is not torch.int64 or target.device != device:
        raise ValueError("target must be an int64 tensor on x's device")
    if device.index != _current_device():
        with torch.cuda.device(device):
            return linear_cross_entropy(x, weight, target, bias, ignore_index, reduction)
    x2 = _matrix(x if x.dim() == 2 else x.reshape(-1, K))
    t = target.reshape(-1)
    t = t if t.is_contiguous() else t.contiguous()
    w = weight if weight.is_contiguous() else weight.contiguous()
    if K % 8 == 0:   # (rows at 16-byte addresses)
        if x2.data_ptr() % 16 or x2.shape[0] > 1 and (x2.stride(0) % 8 or x2.stride(0) >= 2**22):
            x2 = x2.clone(memory_format=torch.contiguous_format)
        if w.data_ptr() % 16:
            w = w.clone()
    b = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or bias is not None and bias.requires_grad):
        loss = _LinearCrossEntropy.apply(x2, w, b, t, int(ignore_index), how)
    else:
        loss = _loss_forward(x2, w, b, t, int(ignore_index), how)
    return loss if how else loss.view(target.shape)


_LINEAR_FORWARD, _LINEAR = torch.nn.Linear.forward, torch.nn.functional.linear


def _watched() -> bool:
    """Whether something sees, replaces or transforms torch's calls: compilation
    and tracing, autocast, dispatch modes, function modes (torch.device's own
    does neither), functorch's transforms, forward-mode differentiation (which
    no_grad leaves on)."""
    if torch.compiler.is_compiling():
        return True
    c = torch._C
    modes = c._len_torch_function_stack()
    return (c._len_torch_dispatch_stack() > 0
            or modes > 0 and any(type(c._get_function_stack_at(i)) is not DeviceContext
                                 for i in range(modes))
            or torch.is_autocast_enabled() or forward_ad._current_level >= 0
            or c._functorch.peek_interpreter_stack() is not None or torch.jit.is_tracing())


def _has_no_hooks(m: torch.nn.Module) -> bool:
    hooks = torch.nn.modules.module
    return not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks
                or m._backward_pre_hooks or hooks._global_forward_hooks
                or hooks._global_forward_pre_hooks or hooks._global_backward_hooks
                or hooks._global_backward_pre_hooks)


def _is_plain_linear(m: torch.nn.Module) -> bool:
    """A torch.nn.Linear whose call is its product and nothing else."""
    return (type(m) is torch.nn.Linear and "forward" not in m.__dict__
            and torch.nn.Linear.forward is _LINEAR_FORWARD
            and torch.nn.functional.linear is _LINEAR and _has_no_hooks(m))


def _project(m: torch.nn.Module, x: torch.Tensor, watched: bool) -> torch.Tensor:
    """m(x), by f3s_linear_f16 where that is the same thing: a plain fp16
    Linear of a contiguous fp16 matrix on its own device, in sizes the kernel
    takes, where nothing watches the call (_watched).  (Called without autograd.)  Below
    64 K rows of more than 128 inputs and outputs the library's tiles are the
    better ones (20,011 x 256 -> 768: 17 against 28 us; -> 128: 8 against 9,
    and half the call's host time)."""
    if (not watched and type(x) is torch.Tensor and x.dim() == 2 and x.is_cuda
            and x.dtype is torch.float16 and x.is_contiguous() and x.shape[0] > 0
            and _is_plain_linear(m)):
        w, b = m.weight, m.bias
        M, K = w.shape
        if (K % 8 == 0 and K <= 256 and M % 32 == 0 and M <= 32768 and x.shape[1] == K
                and (K <= 128 or M <= 128 or x.shape[0] >= 65536)
                and w.dtype is torch.float16 and w.device == x.device and w.is_contiguous()
                and type(w) is torch.nn.Parameter
                and (b is None or (type(b) is torch.nn.Parameter and b.dtype is torch.float16
                                   and b.device == x.device and b.is_contiguous()))
                and (x.data_ptr() | w.data_ptr()) % 16 == 0
                and x.device.index == torch.cuda.current_device()):
            y = torch.empty((x.shape[0], M), dtype=torch.float16, device=x.device)
            check(_lib.hip().f3s_linear_f16(
                x.data_ptr(), w.data_ptr(), b.data_ptr() if b is not None else None,
                y.data_ptr(), x.shape[0], K, M, torch.cuda.current_stream().cuda_stream),
                "f3s_linear_f16")
            return y
    return m(x)


_ATTENTION = TorchGraph.attention


def _is_plain_graph(graph) -> bool:
    """Whether attention_packed stands for graph.attention: not where a
    program brings an attention of its own, in a subclass, on the graph or in
    the place of TorchGraph's."""
    return (isinstance(graph, TorchGraph) and type(graph).attention is _ATTENTION
            and "attention" not in graph.__dict__)


class GraphTransformerLayer(torch.nn.Module):
    """x -> [Q K V] = x W_qkv -> fused edge attention per head -> concat ->
    W_o, forward only.  Compute dtype of the projections is the module's
    (fp16 after .half()); attention accumulates and returns fp32, which is
    cast back to the projection dtype before W_o."""

    def __init__(self, in_dim: int, heads: int = 1, out_dim: int | None = None,
                 bias: bool = True):
        super().__init__()
        self.heads = heads
        self.qkv = torch.nn.Linear(in_dim, 3 * heads * HEAD_DIM, bias=bias)
        self.proj = torch.nn.Linear(heads * HEAD_DIM, out_dim or in_dim, bias=bias)
        self.scale = HEAD_DIM ** -0.5

    @torch.no_grad()
    def forward(self, x: torch.Tensor, graph: TorchGraph) -> torch.Tensor:
        if graph.heads != self.heads:
            raise ValueError("graph was planned for a different head count")
        n = x.shape[0]
        watched = _watched()
        qkv = _project(self.qkv, x, watched).to(torch.float16)
        dtype = self.proj.weight.dtype
        if _is_plain_graph(graph) and graph.takes_packed() and qkv.dim() == 2 \
                and qkv.is_contiguous():
            # the pass reads q, k and v where the projection wrote them, and
            # writes O in the dtype the output projection takes
            o = graph.attention_packed(qkv, self.scale,
                                       dtype if dtype == torch.float16 else torch.float32)
        else:
            qkv = qkv.view(n, 3, self.heads, HEAD_DIM)
            q, k, v = (qkv[:, i].contiguous() for i in range(3))
            o = graph.attention(q, k, v, scale=self.scale)
        return _project(self.proj, o.view(n, self.heads * HEAD_DIM).to(dtype), watched)


_TORCH_ACTIVATIONS = {
    None: lambda z: z, "relu": torch.nn.functional.relu, "gelu": torch.nn.functional.gelu,
    "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh"),
    "silu": torch.nn.functional.silu}


def _dense(m: torch.nn.Module, x: torch.Tensor, watched: bool, activation: str | None = None,
           residual: torch.Tensor | None = None) -> torch.Tensor:
    """activation(m(x)) + residual: linear() where m is a plain Linear of plain tensors
    of a type it takes and nothing watches the call, else torch's own operations."""
    if (not watched and _is_plain_linear(m) and type(x) is torch.Tensor and x.is_cuda
            and type(m.weight) in _PLAIN and type(m.bias) in _PLAIN
            and (residual is None or type(residual) is torch.Tensor)
            and x.dtype in _DTYPES and m.weight.dtype == x.dtype and m.weight.device == x.device
            and (residual is None or residual.dtype == x.dtype)):
        return linear(x, m.weight, m.bias, activation, residual)
    y = _TORCH_ACTIVATIONS[activation](m(x))
    return y if residual is None else y + residual


class DiffGraphTransformerLayer(torch.nn.Module):
    """Differential attention over a graph's edges with its projections, and
    optionally a feed-forward part; trainable.

        o_h = rms_norm(diff_attention(x W_qkv)_h) * (1 - lambda_init)
        y = concat(o) W_o + x                      (residual=True)
        y = activation(y W_up) W_down + y          (ffn_dim given)

    A head's weight is exp(lambda_q1 . lambda_k1) - exp(lambda_q2 . lambda_k2) +
    lambda_init, from four learned vectors.  Two maps of 64 dims and values of
    128 per head, so `heads` heads project to heads * 128 features; the graph has
    to be made for `heads` heads.  Computes in the module's type (float16 or
    bfloat16; a float32 module's attention runs in float16)."""

    def __init__(self, in_dim: int, heads: int = 1, out_dim: int | None = None, bias: bool = True,
                 lambda_init: float = 0.8, residual: bool = True, ffn_dim: int | None = None,
                 activation: str = "gelu", eps: float = 1e-5):
        super().__init__()
        out_dim = out_dim or in_dim
        if residual and out_dim != in_dim:
            raise ValueError("a residual needs out_dim == in_dim")
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {list(_ACTIVATIONS)}")
        self.heads, self.lambda_init, self.residual = heads, float(lambda_init), residual
        self.activation, self.eps, self.scale = activation, eps, HEAD_DIM ** -0.5
        self.qkv = torch.nn.Linear(in_dim, 3 * heads * 2 * HEAD_DIM, bias=bias)
        self.proj = torch.nn.Linear(heads * 2 * HEAD_DIM, out_dim, bias=bias)
        self.norm = torch.nn.Parameter(torch.ones(2 * HEAD_DIM))
        for name in ("lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2"):
            setattr(self, name, torch.nn.Parameter(0.1 * torch.randn(heads, HEAD_DIM)))
        self.up = torch.nn.Linear(out_dim, ffn_dim, bias=bias) if ffn_dim else None
        self.down = torch.nn.Linear(ffn_dim, out_dim, bias=bias) if ffn_dim else None

    def head_weights(self) -> torch.Tensor:
        """lam, float32 [heads]."""
        q1, k1, q2, k2 = (t.float() for t in (self.lambda_q1, self.lambda_k1, self.lambda_q2,
                                              self.lambda_k2))
        return torch.exp((q1 * k1).sum(-1)) - torch.exp((q2 * k2).sum(-1)) + self.lambda_init

    def forward(self, x: torch.Tensor, graph: TorchGraph) -> torch.Tensor:
        if graph.heads != self.heads:
            raise ValueError("graph was planned for a different head count")
        watched = _watched()
        qkv = _dense(self.qkv, x, watched)
        if qkv.dtype not in _DTYPES:
            qkv = qkv.to(torch.float16)
        o = graph.diff_attention_packed(qkv, self.head_weights(), self.scale)
        dtype = self.proj.weight.dtype
        o = torch.nn.functional.rms_norm(o.to(dtype), (2 * HEAD_DIM,),
                                         self.norm * (1.0 - self.lambda_init), self.eps)
        y = _dense(self.proj, o.view(x.shape[0], self.heads * 2 * HEAD_DIM), watched, None,
                   x if self.residual else None)
        if self.up is not None:
            y = _dense(self.down, _dense(self.up, y, watched, self.activation), watched, None, y)
        return y


_NORM_FORWARD, _NORM = torch.nn.LayerNorm.forward, torch.nn.functional.layer_norm


def _norm(m: torch.nn.Module, x: torch.Tensor, watched: bool) -> torch.Tensor:
    """m(x): layer_norm() where m is a plain LayerNorm of plain tensors of types that it
    takes and nothing watches the call, else torch's own."""
    if (not watched and type(m) is torch.nn.LayerNorm and "forward" not in m.__dict__
            and torch.nn.LayerNorm.forward is _NORM_FORWARD
            and torch.nn.functional.layer_norm is _NORM and _has_no_hooks(m)
            and len(m.normalized_shape) == 1 and x.dim() >= 1
            and x.shape[-1] == m.normalized_shape[0] and type(x) is torch.Tensor and x.is_cuda
            and x.dtype in _NORM_DTYPES and type(m.weight) in _PLAIN and type(m.bias) in _PLAIN
            and all(t is None or t.dtype in (x.dtype, torch.float32) and t.device == x.device
                    for t in (m.weight, m.bias))
            and (m.weight is None or m.bias is None or m.weight.dtype == m.bias.dtype)):
        return layer_norm(x, m.weight, m.bias, m.eps)
    return m(x)


class EdgeGraphTransformerLayer(torch.nn.Module):
    """A pre-norm layer of softmax attention over a graph's edges, optionally with a
    feed-forward part; trainable.

        h = edge_attention(norm1(x) W_qkv) W_o + x
        y = activation(norm2(h) W_up) W_down + h      (ffn_dim given)

    cap: scores are capped to cap * tanh(score / cap).  distance: scores are lowered by
    slopes[h] times the distance of the two nodes' `positions` ([n] or [n, 1 to 3]
    float32, given to the call), slopes learned, 1/2, 1/4, .. at first.  `heads` heads
    of 64 dims; the graph has to be made for `heads` heads.  Computes in the module's
    type (float16 or bfloat16; a float32 module's attention runs in float16)."""

    def __init__(self, in_dim: int, heads: int = 1, bias: bool = True, ffn_dim: int | None = None,
                 activation: str = "gelu", cap: float | None = None, distance: bool = False,
                 eps: float = 1e-5):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {list(_ACTIVATIONS)}")
        self.heads, self.activation, self.cap, self.scale = heads, activation, cap, HEAD_DIM ** -0.5
        self.norm1 = torch.nn.LayerNorm(in_dim, eps=eps)
        self.qkv = torch.nn.Linear(in_dim, 3 * heads * HEAD_DIM, bias=bias)
        self.proj = torch.nn.Linear(heads * HEAD_DIM, in_dim, bias=bias)
        self.slopes = (torch.nn.Parameter(0.5 ** torch.arange(1, heads + 1).float())
                       if distance else None)
        self.norm2 = torch.nn.LayerNorm(in_dim, eps=eps) if ffn_dim else None
        self.up = torch.nn.Linear(in_dim, ffn_dim, bias=bias) if ffn_dim else None
        self.down = torch.nn.Linear(ffn_dim, in_dim, bias=bias) if ffn_dim else None

    def forward(self, x: torch.Tensor, graph: TorchGraph,
                positions: torch.Tensor | None = None) -> torch.Tensor:
        if graph.heads != self.heads:
            raise ValueError("graph was planned for a different head count")
        if (positions is None) != (self.slopes is None):
            raise ValueError("positions are for a layer made with distance=True")
        watched = _watched()
        qkv = _dense(self.qkv, _norm(self.norm1, x, watched), watched)
        if qkv.dtype not in _DTYPES:
            qkv = qkv.to(torch.float16)
        o = graph.edge_attention_packed(qkv, self.scale, self.cap, positions,
                                        None if self.slopes is None else self.slopes.float())
        y = _dense(self.proj, o.view(x.shape[0], -1).to(self.proj.weight.dtype), watched, None, x)
        if self.up is not None:
            z = _dense(self.up, _norm(self.norm2, y, watched), watched, self.activation)
            y = _dense(self.down, z, watched, None, y)
        return y


# ------------------------------------------------------------------ operator

def _cuda_i32(t, what: str) -> torch.Tensor:
    """An int32 CUDA copy (or view) of an integer array; int64 input (the
    usual index type of torch graph code) is narrowed after a range check."""
    t = torch.as_tensor(t)
    if t.dtype == torch.int64:
        if t.numel() and (int(t.min()) < -2**31 or int(t.max()) >= 2**31):
            raise ValueError(f"{what} holds values outside the int32 range")
        t = t.to(torch.int32)
    elif t.dtype != torch.int32:
        raise ValueError(f"{what} must hold int32 (or int64) values")
    if not t.is_cuda:
        t = t.to("cuda")
    return t.contiguous()


def to_block_sparse(row_ptr, col_idx, masks: bool = True):
    """convert_csr_to_block_sparse (src/converter.cu:13-44) on the GPU into
    torch tensors: (window_offsets int32 [W + 1], block_col_indices int32
    [T], tile_mask int16 [T, 16] -- bit c of row r of a tile set iff that
    edge exists -- or None).  Two calls of f3s_convert_csr_to_bsf on torch's
    current stream, the count (one host round trip for T), then the fill; or,
    on small graphs, one call for both, whose lists are then views of storage
    for at most four times their entries, or 4 MB more (lists_oversized)."""
    rp = _cuda_i32(row_ptr, "row_ptr")
    ci = _cuda_i32(col_idx, "col_idx")
    n = rp.numel() - 1
    if n < 0:
        raise ValueError("row_ptr must hold n + 1 entries")
    W = (n + 15) // 16
    lib = _lib.hip()
    s = torch.cuda.current_stream().cuda_stream
    offs = torch.empty(W + 1, dtype=torch.int32, device=rp.device)
    T = C.c_int64(0)
    cptr = ci.data_ptr() if ci.numel() else None
    if converts_once(n, ci.numel()):
        most = most_tiles(n, ci.numel())
        bcol = torch.empty(most, dtype=torch.int32, device=rp.device)
        mask = torch.empty((most, 16), dtype=torch.int16, device=rp.device) if masks else None
        check(lib.f3s_convert_csr_to_bsf_once(
            rp.data_ptr(), cptr, n, ci.numel(), offs.data_ptr(), bcol.data_ptr(),
            mask.data_ptr() if masks else None, C.byref(T), s), "f3s_convert_csr_to_bsf_once")
        t = int(T.value)
        bcol, mask = bcol[:t], (mask[:t] if masks else None)
        if lists_oversized(t, most):
            bcol, mask = bcol.clone(), (mask.clone() if masks else None)
        return offs, bcol, mask
    check(lib.f3s_convert_csr_to_bsf(rp.data_ptr(), cptr, n, ci.numel(), offs.data_ptr(), None,
                                     None, C.byref(T), s), "f3s_convert_csr_to_bsf(count)")
    t = int(T.value)
    # at least one element each, so the fill call gets real pointers
    bcol = torch.empty(max(t, 1), dtype=torch.int32, device=rp.device)
    mask = torch.empty((max(t, 1), 16), dtype=torch.int16, device=rp.device) if masks else None
    T2 = C.c_int64(0)
    check(lib.f3s_convert_csr_to_bsf(rp.data_ptr(), cptr, n, ci.numel(), offs.data_ptr(),
                                     bcol.data_ptr(), mask.data_ptr() if masks else None,
                                     C.byref(T2), s), "f3s_convert_csr_to_bsf(fill)")
    return offs, bcol[:t], (mask[:t] if masks else None)


def _check_operands(q, k, v, window_offsets, block_col, tile_mask, window_order):
    if q.dim() != 3 or q.shape[2] != HEAD_DIM:
        raise ValueError(f"q must be [n, H, {HEAD_DIM}]")
    n, H = q.shape[0], q.shape[1]
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dtype != torch.float16 or not t.is_cuda or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous float16 CUDA tensor")
        if tuple(t.shape) != (n, H, HEAD_DIM):
            raise ValueError(f"{name} must have shape {(n, H, HEAD_DIM)}, got {tuple(t.shape)}")
    W = (n + 15) // 16
    for name, t, shape in (("window_offsets", window_offsets, (W + 1,)),
                           ("block_col", block_col, None),
                           ("window_order", window_order, (W,))):
        if t is None:
            if name != "window_order":
                raise ValueError(f"{name} is required")
            continue
        if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous() or t.dim() != 1:
            raise ValueError(f"{name} must be a contiguous 1-d int32 CUDA tensor")
        if shape is not None and tuple(t.shape) != shape:
            raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if tile_mask is not None:
        if (tile_mask.dtype not in (torch.int16, torch.uint16) or not tile_mask.is_cuda
                or not tile_mask.is_contiguous()
                or tuple(tile_mask.shape) != (block_col.shape[0], 16)):
            raise ValueError("tile_mask must be a contiguous [T, 16] int16 CUDA tensor")
    return n, H, W


@torch.library.custom_op("fused3s::attention_fwd", mutates_args=())
def attention_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                  window_offsets: torch.Tensor, block_col: torch.Tensor,
                  tile_mask: torch.Tensor | None, window_order: torch.Tensor | None,
                  scale: float = 1.0) -> torch.Tensor:
    """f3s_attention_fwd (the reference's launch, tests/test_fused_3s_v2.cu:
    124-131, every window whole) on torch tensors and torch's current
    stream: q/k/v [n, H, 64] float16, the block-sparse form of
    to_block_sparse, window_order int32 [W] or None (natural order); a
    tile_mask gives the masked (edge-exact) semantics, None the reference's
    tile-dense one.  Returns O [n, H, 64] float32."""
    if q.requires_grad or k.requires_grad or v.requires_grad:
        raise RuntimeError("the fused pass is forward-only (no autograd)")
    n, H, W = _check_operands(q, k, v, window_offsets, block_col, tile_mask, window_order)
    out = torch.empty((n, H, HEAD_DIM), dtype=torch.float32, device=q.device)
    if n == 0:
        return out
    s = torch.cuda.current_stream(q.device).cuda_stream
    # an empty block_col tensor may have no storage: the C-ABI wants a pointer
    # whenever W > 0, and with T = 0 no tile is read through it
    bptr = block_col.data_ptr() or window_offsets.data_ptr()
    mptr = None
    if tile_mask is not None:
        mptr = tile_mask.data_ptr() or out.data_ptr()
    check(_lib.hip().f3s_attention_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                       window_offsets.data_ptr(), bptr, mptr,
                                       window_order.data_ptr() if window_order is not None
                                       else None, W, n, HEAD_DIM, H, float(scale), s),
          "f3s_attention_fwd")
    return out


@attention_fwd.register_fake
def _attention_fwd_fake(q, k, v, window_offsets, block_col, tile_mask, window_order, scale=1.0):
    return torch.empty(q.shape, dtype=torch.float32, device=q.device)
