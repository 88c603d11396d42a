"""Host-side mirror of ``vkml::Backend`` (include/vkml/backend/api/backend.h:49-125)
over the C ABI: same method names, argument meaning and error behaviour, so code
and tests written against vkML's backend interface read the same here.

Errors cross the C boundary as status codes and are raised as the exception
types vkML maps to Python (bindings/module.cpp:243-250).
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Sequence

import numpy as np

from . import _abi, graph
from .graph import DType, NodeDesc, TensorDesc, pack_nodes


class Error(RuntimeError):
    """vkml::Error"""


class ShapeError(Error):
    pass


class DTypeError(Error):
    pass


class DeviceError(Error):
    pass


class OutOfMemoryError(Error):
    pass


class InternalError(Error):
    pass


_STATUS_EXC = {
    1: ShapeError, 2: DTypeError, 3: DeviceError, 4: IndexError, 5: NotImplementedError,
    6: InternalError, 7: OutOfMemoryError, 8: ValueError, 9: DeviceError,
}

COMPUTE_SYNC = 1
COMPUTE_GRAD_SYNC = 2
GEMM_3XTF32, GEMM_TF32, GEMM_FP32 = 0, 1, 2


class Storage:
    """vkml::Storage (include/vkml/core/storage.h:29-55): an owned device byte
    range. Dropping the last reference returns the block to the backend's cache;
    that is safe while kernels using it are queued (stream-ordered reuse)."""

    def __init__(self, backend: "Backend", data: int, nbytes: int):
        self._backend = backend
        self.data = data
        self.nbytes = nbytes

    def __del__(self):
        b, self._backend = getattr(self, "_backend", None), None
        if b is not None and self.data and b._ctx:
            b._lib.b200_free(b._ctx, self.data)


class Backend:
    """One CUDA device behind vkML's backend interface."""

    def __init__(self, cuda_ordinal: int = 0):
        self._lib = _abi.load()
        if self._lib.b200_abi_version() != 1:
            raise DeviceError("vkml_b200: ABI version mismatch")
        ctx = C.c_void_p()
        rc = self._lib.b200_create(cuda_ordinal, C.byref(ctx))
        if rc != 0:
            raise DeviceError(
                f"vkml_b200: cannot open CUDA device {cuda_ordinal}: "
                f"{self._lib.b200_status_name(rc).decode()} (no CPU fallback exists)")
        self._ctx = ctx
        self.ordinal = cuda_ordinal
        caps = _abi.Caps()
        self._check(self._lib.b200_get_caps(self._ctx, C.byref(caps)), "capabilities")
        self._caps = caps

    # -- describe -----------------------------------------------------------
    @property
    def name(self) -> str:
        return "b200:" + self._caps.name.decode()

    @property
    def device(self) -> str:
        # registered under vkML's "vulkan:N" device slot (include/vkml/core/device.h:9-12)
        return f"vulkan:{self.ordinal}"

    def capabilities(self) -> dict:
        c = self._caps
        return {
            "name": c.name.decode(), "compute_capability": (c.cc_major, c.cc_minor),
            "shader_core_count": c.sm_count, "subgroup_size": c.warp_size,
            "max_workgroup_invocations": c.max_threads_per_block,
            "max_shared_memory_bytes": c.max_shared_memory_bytes,
            "total_memory_bytes": c.total_memory_bytes,
            "min_buffer_alignment": c.min_buffer_alignment,
            "asynchronous": True, "host_accessible_buffers": False, "unified_memory": False,
        }

    # -- memory ---------------------------------------------------------------
    def allocate(self, nbytes: int) -> Storage:
        """Allocator::allocate: zero bytes yields a Storage with null data."""
        ptr = C.c_void_p()
        self._check(self._lib.b200_alloc(self._ctx, nbytes, C.byref(ptr)), "allocate")
        return Storage(self, ptr.value or 0, nbytes)

    # -- compute --------------------------------------------------------------
    def supports(self, node: NodeDesc) -> bool:
        c = node.to_c()
        return bool(self._lib.b200_supports(C.byref(c)))

    def matmul_kernel(self, node: NodeDesc) -> tuple:
        """(kernel, reason) a matmul node would get, taken by itself: fp32_simt, tcgen05_3xtf32 (operand
        planes, or split inside the kernel), tcgen05_3xtf32_stream (streamed operand), tcgen05_3xtf32_direct
        (operands read directly) or tcgen05_3xf16 (half terms)."""
        c = node.to_c()
        name, why = C.create_string_buffer(64), C.create_string_buffer(160)
        self._check(self._lib.b200_matmul_kernel(self._ctx, C.byref(c), name, 64, why, 160), "matmul_kernel")
        return name.value.decode(), why.value.decode()

    def compute(self, nodes: Sequence[NodeDesc], flags: int = 0) -> None:
        """Backend::compute: ordered when this returns, not necessarily finished."""
        self.compute_packed(pack_nodes(nodes), len(nodes), flags)

    def compute_packed(self, packed, n: int, flags: int = 0) -> None:
        self._check(self._lib.b200_compute(self._ctx, packed, n, flags), "compute")

    # -- operators of language-model training ---------------------------------
    # Tensors are DeviceTensor or TensorDesc; results are tensors that the caller made.  Every call is ordered on the
    # backend's stream when it returns, like compute().  `workspace`: a Storage for calls that are captured into a
    # graph of the caller's, which are refused without one; else the context's own scratch is used.
    def embedding(self, table, ids, rows, scale: float = 1.0) -> None:
        """rows[t] = scale * table[ids[t]].  table [V, D], ids of any extents up to rank 2 (I64 or I32), rows
        ids' extents and D; F32 or F16 on either side.  An id outside [0, V) reads as zeros and is an IndexError at
        the next synchronisation."""
        self._check(self._lib.b200_embedding(self._ctx, graph.embedding_args(table, ids, rows, scale)), "embedding")

    def embedding_backward(self, rows_grad, ids, table_grad, scale: float = 1.0, padding_id: int | None = None,
                           accumulate: bool = False, workspace: Storage | None = None) -> None:
        """table_grad[v] = scale * (the sum of rows_grad over the tokens of id v), zeros where there are none; with
        `accumulate` added to what table_grad holds (a tied projection's gradient).  Tokens of `padding_id` are left
        out.  Sums are held in F32, in an order that the ids alone decide."""
        ws, nbytes = (workspace.data, workspace.nbytes) if workspace is not None else (0, 0)
        self._check(self._lib.b200_embedding_backward(self._ctx, graph.embedding_args(
            table_grad, ids, rows_grad, scale, graph.ACCUMULATE if accumulate else 0,
            -1 if padding_id is None else padding_id, ws, nbytes)), "embedding_backward")

    def embedding_backward_workspace(self, rows_grad, ids, table_grad) -> int:
        """Bytes of a workspace for embedding_backward with these tensors."""
        n = C.c_size_t(0)
        self._check(self._lib.b200_embedding_backward_workspace(
            graph.embedding_args(table_grad, ids, rows_grad, 1.0), C.byref(n)), "embedding_backward_workspace")
        return n.value

    def block_norm(self, residual, branch, *, out=None, normed=None, stats=None, post_weight=None, post_bias=None,
                   gate=None, pre_weight=None, pre_bias=None, residual_scale: float = 1.0, branch_scale: float = 1.0,
                   kind: str = "rms", eps: float = 1e-5, post_norm: bool = True) -> None:
        """out = residual_scale * residual + branch_scale * gate * (N(branch) * post_weight + post_bias);
        normed = N(out) * pre_weight + pre_bias: the norm behind a block, its gate, the sum with the residual
        stream and the norm in front of the next block.  residual or branch may be None, and so may out or normed
        (no norm in front).  `post_norm=False`: the branch as it is.  kind: "rms" or "layer".  stats [rows, 4] F32 is
        what block_norm_backward needs."""
        if branch is None:
            post_norm = False
        self._check(self._lib.b200_block_norm(self._ctx, graph.block_norm_args(
            (residual, branch, out, normed, stats, post_weight, post_bias, pre_weight, pre_bias, gate),
            residual_scale, branch_scale, eps, self._norm_kind(kind), graph.NORM_POST if post_norm else 0)), "block_norm")

    @staticmethod
    def _norm_kind(kind: str) -> int:
        if kind not in graph.NORM_KINDS:
            raise ValueError(f"block_norm: unknown kind of norm {kind!r}")
        return graph.NORM_KINDS[kind]

    def _block_norm_grad_args(self, out, branch, stats, *, out_grad=None, normed_grad=None, residual_grad=None,
                              branch_grad=None, post_weight=None, post_bias=None, gate=None, pre_weight=None,
                              post_weight_grad=None, post_bias_grad=None, gate_grad=None, pre_weight_grad=None,
                              pre_bias_grad=None, residual_scale=1.0, branch_scale=1.0, kind="rms", post_norm=True,
                              workspace=None) -> bytes:
        ws, nbytes = (workspace.data, workspace.nbytes) if workspace is not None else (0, 0)
        if branch is None:
            post_norm = False
        return graph.block_norm_grad_args(
            (out, branch, stats, out_grad, normed_grad, post_weight, post_bias, gate, pre_weight, residual_grad, branch_grad,
             post_weight_grad, post_bias_grad, pre_weight_grad, pre_bias_grad, gate_grad),
            residual_scale, branch_scale, self._norm_kind(kind), graph.NORM_POST if post_norm else 0, ws, nbytes)

    def block_norm_backward(self, out, branch, stats, **options) -> None:
        """Gradients of block_norm from out_grad and normed_grad (either may be None: zero), with out and stats as the forward
        call left them: residual_grad, branch_grad, post_weight_grad, post_bias_grad, gate_grad, pre_weight_grad and
        pre_bias_grad, each where a tensor is given.  The other options are those of the forward call, and workspace."""
        self._check(self._lib.b200_block_norm_backward(
            self._ctx, self._block_norm_grad_args(out, branch, stats, **options)), "block_norm_backward")

    def block_norm_backward_workspace(self, out, branch, stats, **options) -> int:
        """Bytes of a workspace for block_norm_backward with these tensors and options."""
        n = C.c_size_t(0)
        self._check(self._lib.b200_block_norm_backward_workspace(
            self._block_norm_grad_args(out, branch, stats, **options), C.byref(n)), "block_norm_backward_workspace")
        return n.value

    def distill_loss(self, logits, teacher_ids, teacher_logits, losses, *, labels=None, stats=None, grad=None,
                     losses_grad=None, temperature: float = 1.0, hard_weight: float = 0.0,
                     grad_scale: float = 1.0) -> None:
        """losses = (1 - hard_weight) * T^2 * KL(softmax(teacher_logits / T) || softmax(logits / T) at teacher_ids)
        + hard_weight * cross-entropy on labels, one F32 for each row.  Ids or labels below 0 are no entry.  With `grad`
        the logits' gradient too, grad_scale * losses_grad * d loss / d logits, from the same reading of the logits (it
        may lie on them).  stats [rows, 4] F32 is what distill_loss_backward needs."""
        self._check(self._lib.b200_distill_loss(self._ctx, graph.distill_args(
            (logits, teacher_ids, teacher_logits, labels, losses, stats, losses_grad, grad), temperature, hard_weight,
            grad_scale)), "distill_loss")

    def distill_loss_backward(self, logits, teacher_ids, teacher_logits, stats, grad, *, labels=None, losses_grad=None,
                              temperature: float = 1.0, hard_weight: float = 0.0, grad_scale: float = 1.0) -> None:
        """The logits' gradient alone, with stats as distill_loss left it; options as there."""
        self._check(self._lib.b200_distill_loss_backward(self._ctx, graph.distill_args(
            (logits, teacher_ids, teacher_logits, labels, None, stats, losses_grad, grad), temperature, hard_weight,
            grad_scale)), "distill_loss_backward")

    def gated_recurrence(self, x, gate, out, *, initial=None, final=None, states=None, lengths=None, kind: str = "sigmoid") -> None:
        """out[t] = h = a[t] * h + b[t] along the axis in front of the last, each channel by itself.  kind "sigmoid":
        a = sigmoid(gate), b = (1 - a) * x; "exp": a = exp(gate), b = x.  x, gate and out [L, D] or [B, L, D]; `initial`
        and `final` [D] or [B, D] F32 are h in front of the first step (None: zeros) and behind the last, and may be one
        tensor: that is how a sequence is continued token by token.  `lengths` [B]: steps of each sequence; behind them out is zeros.  `states`
        [.., ceil(L / 16), D] F32 is what gated_recurrence_backward needs."""
        self._check(self._lib.b200_gated_recurrence(self._ctx, graph.recurrence_args(
            (x, gate, initial, lengths, out, final, states), self._gate_kind(kind))), "gated_recurrence")

    @staticmethod
    def _gate_kind(kind: str) -> int:
        if kind not in graph.GATE_KINDS:
            raise ValueError(f"gated_recurrence: unknown kind of gates {kind!r}")
        return graph.GATE_KINDS[kind]

    def gated_recurrence_backward(self, x, gate, states, *, out_grad=None, final_grad=None, x_grad=None, gate_grad=None,
                                  initial_grad=None, lengths=None, kind: str = "sigmoid") -> None:
        """Gradients of gated_recurrence from out_grad and final_grad (either may be None: zero), with states as the forward call left
        them: x_grad, gate_grad and initial_grad, each where a tensor is given."""
        self._check(self._lib.b200_gated_recurrence_backward(self._ctx, graph.recurrence_args(
            (x, gate, lengths, states, out_grad, final_grad, x_grad, gate_grad, initial_grad), self._gate_kind(kind))),
            "gated_recurrence_backward")

    def token_logprobs(self, logits, tokens=None, logprobs=None, *, entropies=None, stats=None, top_ids=None, top_logprobs=None,
                       temperature: float = 1.0) -> None:
        """logprobs = log softmax(logits / T) at tokens, one F32 for each row (0 where the token is below 0); entropies of the same
        distributions; top_ids [.., K] (I32 or I64) the columns of the K <= 128 largest logits, the largest first (equal ones: the lowest
        column), and top_logprobs [.., K] F32 their log probabilities -- what distill_loss reads as a teacher's.  Each where a tensor is given.
        stats [rows, 4] F32 is what token_logprobs_backward needs."""
        self._check(self._lib.b200_token_logprobs(self._ctx, graph.logprobs_args(
            (logits, tokens, logprobs, entropies, stats, top_ids, top_logprobs, None, None, None), temperature, 1.0)), "token_logprobs")

    def token_logprobs_backward(self, logits, tokens, stats, grad, *, logprobs_grad=None, entropies_grad=None,
                                temperature: float = 1.0, grad_scale: float = 1.0) -> None:
        """The logits' gradient from those of logprobs and entropies (either may be None: zero), times grad_scale, with stats as
        token_logprobs left them; grad may lie on logits."""
        self._check(self._lib.b200_token_logprobs_backward(self._ctx, graph.logprobs_args(
            (logits, tokens, None, None, stats, None, None, logprobs_grad, entropies_grad, grad), temperature, grad_scale)),
            "token_logprobs_backward")

    def adamw(self, tensors, *, lr, step, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8, grad_scale=1.0,
              seed: int = 0) -> None:
        """One AdamW step over all tensors: a sequence of AdamWTensor, or what adamw_table() made of one, once for all steps (a sequence is
        described anew in every call, some 3 us a tensor, which for a small model is more than the step itself).  States in
        F32, or in 8 bits with a scale to 256 elements, rounded up or down by bits of seed and step.  lr, step (from 1 on) and grad_scale are
        numbers, or one-element tensors on the device (F32, I64, F32) for a step that is captured once: where grad_scale is not finite there,
        or step below 1, nothing changes."""
        table = tensors if isinstance(tensors, graph.AdamWTable) else graph.adamw_table(tensors)
        args, keep = graph.adamw_args(table, lr, step, beta1, beta2, eps, grad_scale, seed)
        self._check(self._lib.b200_adamw(self._ctx, args), "adamw")
        del keep

    # -- copies ---------------------------------------------------------------
    def copy_from_host(self, dst: Storage, dst_offset: int, src, nbytes: int | None = None) -> None:
        buf = np.ascontiguousarray(src) if not isinstance(src, int) else None
        n = nbytes if nbytes is not None else buf.nbytes
        if n == 0:
            return
        if dst_offset < 0 or dst_offset + n > dst.nbytes:
            raise IndexError(f"copy_from_host writes {n} bytes at offset {dst_offset} into a "
                             f"{dst.nbytes}-byte storage")
        ptr = src if isinstance(src, int) else buf.ctypes.data
        self._check(self._lib.b200_copy_from_host(self._ctx, dst.data + dst_offset, ptr, n),
                    "copy_from_host")

    def copy_to_host(self, dst: np.ndarray, src: Storage, src_offset: int, nbytes: int | None = None) -> None:
        n = nbytes if nbytes is not None else dst.nbytes
        if n == 0:
            return
        if src_offset < 0 or src_offset + n > src.nbytes:
            raise IndexError(f"copy_to_host reads {n} bytes at offset {src_offset} from a "
                             f"{src.nbytes}-byte storage")
        assert dst.flags["C_CONTIGUOUS"]
        self._check(self._lib.b200_copy_to_host(self._ctx, dst.ctypes.data, src.data + src_offset, n),
                    "copy_to_host")

    def copy_device_to_device(self, copies: Sequence[tuple]) -> None:
        """copies: (dst Storage, dst_offset, src Storage, src_offset, nbytes); disjoint ranges."""
        words = []
        for d, doff, s, soff, n in copies:
            if doff < 0 or doff + n > d.nbytes or soff < 0 or soff + n > s.nbytes:
                raise IndexError("copy_device_to_device range exceeds a storage")
            words += (d.data + doff, s.data + soff, n)
        if not words:
            return
        arr = (_abi.Copy * len(copies)).from_buffer_copy(struct.pack("<%dQ" % len(words), *words))
        self._check(self._lib.b200_copy_device_to_device(self._ctx, arr, len(copies)),
                    "copy_device_to_device")

    def synchronize(self) -> None:
        self._check(self._lib.b200_synchronize(self._ctx), "synchronize")

    # -- policy / introspection -------------------------------------------------
    def set_gemm_precision(self, precision: int) -> None:
        self._check(self._lib.b200_set_gemm_precision(self._ctx, precision), "set_gemm_precision")

    def stats(self) -> dict:
        s = _abi.Stats()
        self._check(self._lib.b200_get_stats(self._ctx, C.byref(s)), "stats")
        return {name: getattr(s, name) for name, _ in s._fields_}

    def set_profiling(self, enabled: bool) -> None:
        """Bracket every kernel launch with device timestamps (VulkanBackend::set_profiling)."""
        self._check(self._lib.b200_profile_enable(self._ctx, 1 if enabled else 0), "profile_enable")

    def last_profile(self, capacity: int = 65536) -> list:
        """[(label, gpu_ms)] in launch order since the last read; synchronises."""
        buf = (_abi.ProfileRecord * capacity)()
        n = C.c_size_t(0)
        self._check(self._lib.b200_profile_read(self._ctx, buf, capacity, C.byref(n)), "profile_read")
        return [(buf[i].label.decode(), float(buf[i].ms)) for i in range(n.value)]

    def span_graph_stats(self) -> tuple:
        """(spans served by launching a kept CUDA graph, graphs captured) since the context was created."""
        hits, captures = C.c_uint64(0), C.c_uint64(0)
        self._check(self._lib.b200_span_graph_stats(self._ctx, C.byref(hits), C.byref(captures)), "span_graph_stats")
        return int(hits.value), int(captures.value)

    def timer_begin(self) -> None:
        self._check(self._lib.b200_timer_begin(self._ctx), "timer_begin")

    def timer_end(self) -> float:
        """Device milliseconds since timer_begin, on the context's stream; synchronises."""
        ms = C.c_float(0)
        self._check(self._lib.b200_timer_end(self._ctx, C.byref(ms)), "timer_end")
        return float(ms.value)

    def alloc_host(self, nbytes: int) -> np.ndarray:
        """Page-locked host bytes as a uint8 array (freed with free_host)."""
        ptr = C.c_void_p()
        self._check(self._lib.b200_alloc_host(self._ctx, nbytes, C.byref(ptr)), "alloc_host")
        arr = np.ctypeslib.as_array((C.c_uint8 * nbytes).from_address(ptr.value))
        self._pinned = getattr(self, "_pinned", {})
        self._pinned[arr.ctypes.data] = ptr.value
        return arr

    def free_host(self, arr: np.ndarray) -> None:
        ptr = getattr(self, "_pinned", {}).pop(arr.ctypes.data, None)
        if ptr is not None:
            self._check(self._lib.b200_free_host(self._ctx, ptr), "free_host")

    def trim(self) -> None:
        self._check(self._lib.b200_trim(self._ctx), "trim")

    @property
    def stream(self) -> int:
        return self._lib.b200_stream(self._ctx) or 0

    # -- data parallel ----------------------------------------------------------
    def dist_unique_id(self) -> bytes:
        buf = C.create_string_buffer(_abi.UNIQUE_ID_BYTES)
        self._check(self._lib.b200_dist_unique_id(buf), "dist_unique_id")
        return buf.raw

    def dist_init(self, rank: int, world: int, unique_id: bytes, timeout_ms: int | None = None) -> None:
        """Join a data-parallel job.  With `timeout_ms`, ranks that do not all arrive in time end
        the call with DeviceError (timeout) and an aborted communicator instead of blocking."""
        buf = C.create_string_buffer(unique_id, _abi.UNIQUE_ID_BYTES)
        if timeout_ms is None:
            self._check(self._lib.b200_dist_init(self._ctx, rank, world, buf), "dist_init")
        else:
            self._check(self._lib.b200_dist_init_deadline(self._ctx, rank, world, buf, timeout_ms), "dist_init")

    def dist_all_reduce_mean(self, data: int, count: int) -> None:
        self._check(self._lib.b200_dist_all_reduce_mean(self._ctx, data, count), "all_reduce")

    def dist_wait(self) -> None:
        self._check(self._lib.b200_dist_wait(self._ctx), "dist_wait")

    def dist_mark_grad(self, data: int, count: int) -> None:
        self._check(self._lib.b200_dist_mark_grad(self._ctx, data, count), "dist_mark_grad")

    def dist_clear_grads(self) -> None:
        self._check(self._lib.b200_dist_clear_grads(self._ctx), "dist_clear_grads")

    def close(self) -> None:
        if self._ctx:
            self._lib.b200_destroy(self._ctx)
            self._ctx = None

    # -- helpers ----------------------------------------------------------------
    def _check(self, rc: int, where: str) -> None:
        if rc == 0:
            return
        detail = self._lib.b200_last_error(self._ctx) if self._ctx else b""
        msg = f"b200 backend: {where}: {self._lib.b200_status_name(rc).decode()}"
        if detail:
            msg += ": " + detail.decode(errors="replace")
        raise _STATUS_EXC.get(rc, InternalError)(msg)


class DeviceTensor:
    """A strided view over a Storage: the fields of a vkML node the backend reads
    (shape with byte strides, dtype, storage, storage_offset; node.h:69-157)."""

    def __init__(self, backend: Backend, storage: Storage, dims, strides, dtype: DType, offset: int = 0):
        self.backend = backend
        self.storage = storage
        self.dims = tuple(int(d) for d in dims)
        self.strides = tuple(int(s) for s in strides)
        self.dtype = DType(dtype)
        self.offset = offset

    # creation
    @staticmethod
    def empty(backend: Backend, dims, dtype: DType = DType.F32) -> "DeviceTensor":
        desc = TensorDesc.contiguous(0, dims, DType(dtype))
        return DeviceTensor(backend, backend.allocate(desc.nbytes), desc.dims, desc.strides, dtype)

    @staticmethod
    def from_host(backend: Backend, array: np.ndarray) -> "DeviceTensor":
        a = np.ascontiguousarray(array)
        t = DeviceTensor.empty(backend, a.shape, DType.of(a.dtype))
        backend.copy_from_host(t.storage, 0, a)
        return t

    @property
    def numel(self) -> int:
        n = 1
        for d in self.dims:
            n *= d
        return n

    @property
    def desc(self) -> TensorDesc:
        return TensorDesc((self.storage.data + self.offset) if self.storage.data else 0,
                          self.dims, self.strides, self.dtype)

    # views (no kernels: the executor resolves them by aliasing, backend.h:34-45)
    def transpose(self, a: int, b: int) -> "DeviceTensor":
        d, s = list(self.dims), list(self.strides)
        d[a], d[b] = d[b], d[a]
        s[a], s[b] = s[b], s[a]
        return DeviceTensor(self.backend, self.storage, d, s, self.dtype, self.offset)

    def reshape(self, dims) -> "DeviceTensor":
        desc = TensorDesc.contiguous(0, dims, self.dtype)
        assert self.is_contiguous() and desc.numel == self.numel
        return DeviceTensor(self.backend, self.storage, desc.dims, desc.strides, self.dtype, self.offset)

    def broadcast_to(self, dims) -> "DeviceTensor":
        dims = tuple(dims)
        pad = len(dims) - len(self.dims)
        d = (1,) * pad + self.dims
        s = (0,) * pad + self.strides
        out_s = []
        for have, want, st in zip(d, dims, s):
            if have == want:
                out_s.append(st)
            else:
                assert have == 1
                out_s.append(0)
        return DeviceTensor(self.backend, self.storage, dims, out_s, self.dtype, self.offset)

    def is_contiguous(self) -> bool:
        if self.numel == 0:
            return True
        expected = self.dtype.itemsize
        for d, s in zip(reversed(self.dims), reversed(self.strides)):
            if d == 1:
                continue
            if s != expected:
                return False
            expected *= d
        return True

    def numpy(self) -> np.ndarray:
        """Synchronising read of a CONTIGUOUS tensor (Tensor::to_host makes a
        Contiguous node first when strided; callers here do the same)."""
        assert self.is_contiguous()
        out = np.empty(self.dims, dtype=self.dtype.numpy)
        self.backend.copy_to_host(out, self.storage, self.offset, out.nbytes)
        return out
