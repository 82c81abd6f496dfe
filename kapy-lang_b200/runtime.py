"""Host-side runtime: a `Handle` per GPU that turns torch tensors (device memory
and streams are torch's job) into the descriptors of ``include/kapyb.h`` and
calls the C ABI.  Errors come back as the exception classes the reference's
bindings raise: ``ValueError`` for verifier-style rejections (the reference
raises ``std::invalid_argument`` / fails ``verify()``), ``RuntimeError`` for
everything else (``std::runtime_error("pass manager run failed")``,
python/src/passes.cc:72-75).
"""
from __future__ import annotations

import ctypes as C
import os
from typing import Optional, Sequence

from . import _abi as abi


class KapybError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"kapyb status {status}: {message}")
        self.status = status


class KapybTimeout(KapybError):
    pass


def _torch():
    import torch
    return torch


_I32 = 2 ** 31 - 1
_codes: dict = {}
_Tensor2d = abi.Tensor2d  # what a constructor leaves out is zero


def _current_stream(device: int) -> int:
    """torch's current stream on `device`, without the Stream object where torch can."""
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device) if raw is not None else torch.cuda.current_stream(device).cuda_stream


def dtype_code(dt) -> int:
    code = _codes.get(dt)
    if code is None:
        code = _codes[dt] = _dtype_code(dt)
    return code


def _dtype_code(dt) -> int:
    torch = _torch()
    if dt == torch.float16:
        return abi.F16
    if dt == torch.bfloat16:
        return abi.BF16
    if dt == torch.float32:
        return abi.F32
    if dt == torch.float8_e4m3fn:
        return abi.F8E4M3
    if dt == torch.float8_e5m2:
        return abi.F8E5M2
    raise ValueError(f"unsupported element type {dt}")


def torch_dtype(code: int):
    torch = _torch()
    return {abi.F16: torch.float16, abi.BF16: torch.bfloat16, abi.F32: torch.float32,
            abi.F8E4M3: torch.float8_e4m3fn, abi.F8E5M2: torch.float8_e5m2}[code]


def tensor2d(t, padding: int = abi.PAD_ZERO, cache: int = 0) -> abi.Tensor2d:
    """kapy.mk_global over a 2-D torch tensor (any strides that fit i32).  `cache`:
    abi.cache_hints(...) of the ld_global / st_global that touches the tensor."""
    if t.dim() != 2:
        raise ValueError("kapy tensors are rank 2")
    s0, s1 = t.stride()
    for v in (t.shape[0], t.shape[1], s0, s1):
        if v >= 2 ** 31:
            raise ValueError("sizes and strides must fit i32")
    return abi.Tensor2d(t.data_ptr(), 0, t.shape[0], t.shape[1], s0, s1, dtype_code(t.dtype),
                        padding, int(cache), 0)


def matmul_plan(m: int, n: int, k: int, *, dtype=abi.BF16, rhs_dtype=None, out_dtype=None,
                lhs_strides=None, rhs_strides=None, out_strides=None, batch: int = 1,
                sm_count: int = 148, align: int = 256, handle=None) -> str:
    """Text of kapyb_matmul_plan for an [m,k] x [k,n] problem described by shape,
    strides (elements; row-major by default) and the byte alignment of its base
    addresses.  Needs no GPU unless a handle is given."""
    lib = abi.load()
    rhs_dtype = dtype if rhs_dtype is None else rhs_dtype
    out_dtype = dtype if out_dtype is None else out_dtype

    def desc(rows, cols, strides, dt):
        s0, s1 = strides if strides is not None else (cols, 1)
        return abi.Tensor2d(align, 0, rows, cols, s0, s1, dt, abi.PAD_ZERO)

    tl, tr, to = desc(m, k, lhs_strides, dtype), desc(k, n, rhs_strides, rhs_dtype), \
        desc(m, n, out_strides, out_dtype)
    buf = C.create_string_buffer(2048)
    st = lib.kapyb_matmul_plan(handle._h if handle is not None else None,
                               0 if handle is not None else int(sm_count), C.byref(tl),
                               C.byref(tr), C.byref(to), int(batch), buf, len(buf))
    if st != abi.OK:
        msg = lib.kapyb_last_error_string(handle._h if handle is not None else None).decode()
        if st == abi.INVALID_ARG:
            raise ValueError(msg)
        raise KapybError(st, msg)
    return buf.value.decode()


_DTYPE_NAMES = {abi.F16: "f16", abi.BF16: "bf16", abi.F32: "f32", abi.F8E4M3: "f8E4M3",
                abi.F8E5M2: "f8E5M2"}


def tuning_load(path: str) -> int:
    """Adds the tuned dispatch choices of a file to the process-wide table."""
    n = C.c_int32(0)
    lib = abi.load()
    st = lib.kapyb_tuning_load(os.fsencode(path), C.byref(n))
    if st != abi.OK:
        raise ValueError(lib.kapyb_last_error_string(None).decode())
    return n.value


def tuning_clear() -> None:
    abi.load().kapyb_tuning_clear()


def tune_matmul(handle, lhs, rhs, out=None, *, file: Optional[str] = None, iters: int = 10,
                candidates: Optional[Sequence[str]] = None, **epilogue):
    """Times the kernel families on this very problem (device tensors, 2-D or
    batched 3-D) and returns (best path, {path: seconds}).  With `file`, appends
    the winner as a line kapyb_tuning_load understands."""
    torch = _torch()
    batched = lhs.dim() == 3
    m, k = lhs.shape[-2], lhs.shape[-1]
    n = rhs.shape[-1]
    if candidates is None:
        candidates = ["auto", "1cta:64", "1cta:128", "1cta:256", "2cta:128", "2cta:256", "2cta:512"]
        if m <= 64 and not batched:
            candidates.append("skinny")
    if out is None:
        out = torch.empty(lhs.shape[:-1] + (n,), device=lhs.device,
                          dtype=torch.bfloat16 if lhs.dtype.itemsize == 1 else lhs.dtype)
    times = {}
    # what the dispatcher's own choice computes: a forced family has to reproduce it
    handle.set_matmul_path("auto")
    handle.matmul(lhs, rhs, out, **epilogue)
    handle.check()
    want = out.clone()
    try:
        for path in candidates:
            try:
                handle.set_matmul_path(path)
                out.zero_()
                for _ in range(3):
                    handle.matmul(lhs, rhs, out, **epilogue)
                handle.check()
            except (KapybError, ValueError):
                continue  # this family does not take the problem
            # families differ in summation order only: a candidate whose result is off
            # by more than that is broken for this problem and must not win
            d = (out.float() - want.float()).abs().max().item()
            scale = want.float().abs().max().item() or 1.0
            if not (d <= 2e-2 * scale):
                continue
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record()
            for _ in range(iters):
                handle.matmul(lhs, rhs, out, **epilogue)
            e1.record()
            e1.synchronize()
            times[path] = e0.elapsed_time(e1) * 1e-3 / iters
    finally:
        handle.set_matmul_path("auto")
    best = min(times, key=times.get)
    if file is not None and best != "auto":
        la, lb = (lhs[0], rhs[0]) if batched else (lhs, rhs)
        lo = out[0] if batched else out
        # The table is keyed by the problem as the kernel sees it.  An output with
        # its unit stride on axis 0 is computed as the transposed problem
        # (C^T = B^T . A^T): M and N swap, and so do the operands and their majors.
        a_k = la.stride(1) == 1 or k == 1
        b_n = lb.stride(1) == 1 or n == 1
        if lo.stride(1) != 1 and lo.stride(0) == 1:
            m, n = n, m
            a_k, b_n = (lb.stride(0) == 1 or k == 1), (la.stride(0) == 1 or n == 1)
        amaj = "k" if a_k else "mn"
        bmaj = "mn" if b_n else "k"
        with open(file, "a") as f:
            f.write(f"{m} {n} {k} {lhs.shape[0] if batched else 1} {_DTYPE_NAMES[dtype_code(lhs.dtype)]} "
                    f"{amaj} {bmaj} {best}  # {times[best] * 1e6:.1f} us, auto {times.get('auto', 0) * 1e6:.1f} us\n")
    return best, times


class Handle:
    """One per (thread, GPU).  Owns the library context; tensors stay the caller's."""

    def __init__(self, device: int = 0):
        self._lib = abi.load()
        self._h = C.c_void_p()
        st = self._lib.kapyb_create(C.byref(self._h), int(device))
        if st != abi.OK:
            msg = self._lib.kapyb_last_error_string(None).decode()
            raise KapybError(st, msg)
        self.device = int(device)
        self._t = _torch()
        self._torch_device = self._t.device("cuda", self.device)

    def close(self):
        if getattr(self, "_h", None) is not None and self._h:
            self._lib.kapyb_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ------------------------------------------------------------ utilities
    def _raise(self, st: int):
        msg = self._lib.kapyb_last_error_string(self._h).decode()
        if st == abi.INVALID_ARG:
            raise ValueError(msg)
        if st == abi.TIMEOUT:
            raise KapybTimeout(st, msg)
        raise KapybError(st, msg)

    def _stream(self, stream=None) -> C.c_void_p:
        if stream is None:
            stream = _torch().cuda.current_stream(self.device)
        return C.c_void_p(getattr(stream, "cuda_stream", stream))

    def check(self, stream=None):
        """Synchronises the stream and raises if a kernel reported a timeout."""
        st = self._lib.kapyb_check(self._h, self._stream(stream))
        if st != abi.OK:
            self._raise(st)

    def reserve_workspace(self, nbytes: int):
        st = self._lib.kapyb_reserve_workspace(self._h, int(nbytes))
        if st != abi.OK:
            self._raise(st)

    @property
    def last_kernel(self) -> str:
        return self._lib.kapyb_last_kernel(self._h).decode()

    @property
    def launch_count(self) -> int:
        return int(self._lib.kapyb_launch_count(self._h))

    def probe_read(self, n: int = 2, stream=None):
        """Probe words of the last matmul run with debug bit 7 (":d128")."""
        words = (C.c_uint32 * 14)()
        st = self._lib.kapyb_probe_read(self._h, self._stream(stream), words, n)
        if st != abi.OK:
            self._raise(st)
        return [int(w) for w in words[:n]]

    def probe_clock(self, stream=None):
        """(cycles, nanoseconds) of the last matmul run with debug bit 7 (":d128")."""
        cyc, ns = self.probe_read(2, stream)
        return cyc, ns

    def set_matmul_path(self, name: str):
        st = self._lib.kapyb_set_matmul_path(self._h, name.encode())
        if st != abi.OK:
            self._raise(st)

    def _epilogue(self, alpha, bias, bias_axis, activation, rounding):
        ep = abi.Epilogue(float(alpha), None, abi.F32, int(bias_axis), int(activation),
                          int(rounding))
        if bias is not None:
            if not bias.is_contiguous():
                raise ValueError("bias must be contiguous")
            ep.bias = bias.data_ptr()
            ep.bias_dtype = dtype_code(bias.dtype)
        return ep

    # --------------------------------------------------------------- matmul
    def matmul(self, lhs, rhs, out=None, *, acc=None, alpha: float = 1.0, bias=None,
               bias_axis: int = 1, activation: int = abi.ACT_NONE, rounding: int = abi.RN,
               out_dtype=None, impl_way: int = abi.MMA_ANY, stream=None,
               cache=(0, 0, 0)):
        """kapy.matmul at whole-problem scope; 3-D operands run as a batch.  `cache`:
        abi.cache_hints(...) for lhs, rhs and out (their eviction priority becomes the
        L2 policy of the tile loads / stores)."""
        torch = _torch()
        if lhs.dim() == 3:
            return self._matmul_batched(lhs, rhs, out, alpha=alpha, bias=bias, bias_axis=bias_axis,
                                        activation=activation, rounding=rounding,
                                        out_dtype=out_dtype, impl_way=impl_way, stream=stream)
        if out is None:
            out = torch.empty((lhs.shape[0], rhs.shape[1]), device=lhs.device,
                              dtype=out_dtype or lhs.dtype)
        tl, tr, to = tensor2d(lhs, cache=cache[0]), tensor2d(rhs, cache=cache[1]), \
            tensor2d(out, cache=cache[2])
        ta = tensor2d(acc) if acc is not None else None
        ep = self._epilogue(alpha, bias, bias_axis, activation, rounding)
        st = self._lib.kapyb_matmul(self._h, C.byref(tl), C.byref(tr),
                                    C.byref(ta) if ta is not None else None, C.byref(to),
                                    C.byref(ep), impl_way, self._stream(stream))
        if st != abi.OK:
            self._raise(st)
        return out

    def matmul_reduce(self, lhs, rhs, axis: int, out=None, reduced=None, *, alpha: float = 1.0,
                      bias=None, bias_axis: int = 1, activation: int = abi.ACT_NONE,
                      rounding: int = abi.RN, out_dtype=None, combiner: int = abi.RED_ADD,
                      impl_way: int = abi.MMA_ANY, stream=None):
        """matmul whose epilogue also sums its f32 result along `axis` (kapy.reduce
        with an addf lambda on the accumulator tile).  Returns (out, reduced)."""
        torch = _torch()
        if out is None:
            out = torch.empty((lhs.shape[0], rhs.shape[1]), device=lhs.device,
                              dtype=out_dtype or lhs.dtype)
        if reduced is None:
            shape = (1, rhs.shape[1]) if axis == 0 else (lhs.shape[0], 1)
            reduced = torch.empty(shape, device=lhs.device, dtype=torch.float32)
        tl, tr, to, td = tensor2d(lhs), tensor2d(rhs), tensor2d(out), tensor2d(reduced)
        ep = self._epilogue(alpha, bias, bias_axis, activation, rounding)
        st = self._lib.kapyb_matmul_reduce(self._h, C.byref(tl), C.byref(tr), C.byref(to),
                                           C.byref(td), int(axis), int(combiner), C.byref(ep),
                                           impl_way, self._stream(stream))
        if st != abi.OK:
            self._raise(st)
        return out, reduced

    def _matmul_batched(self, lhs, rhs, out, *, alpha, bias, bias_axis, activation, rounding,
                        out_dtype, impl_way, stream):
        torch = _torch()
        if rhs.dim() != 3 or rhs.shape[0] != lhs.shape[0]:
            raise ValueError("batched matmul needs [B,M,K] and [B,K,N]")
        B = lhs.shape[0]
        if out is None:
            out = torch.empty((B, lhs.shape[1], rhs.shape[2]), device=lhs.device,
                              dtype=out_dtype or lhs.dtype)
        tl, tr, to = tensor2d(lhs[0]), tensor2d(rhs[0]), tensor2d(out[0])
        ep = self._epilogue(alpha, bias, bias_axis, activation, rounding)
        st = self._lib.kapyb_matmul_batched(self._h, C.byref(tl), C.byref(tr), C.byref(to), B,
                                            lhs.stride(0), rhs.stride(0), out.stride(0),
                                            C.byref(ep), impl_way, self._stream(stream))
        if st != abi.OK:
            self._raise(st)
        return out

    def matmul_host(self, lhs, rhs, out, *, alpha: float = 1.0, bias=None, bias_axis: int = 1,
                    activation: int = abi.ACT_NONE, rounding: int = abi.RN,
                    impl_way: int = abi.MMA_ANY, stream=None):
        """Same call on CPU tensors (pinned or pageable): copies in, computes on
        the GPU, copies `out` back, returns when it has landed."""
        for t in (lhs, rhs, out):
            if t.is_cuda:
                raise ValueError("matmul_host takes host tensors")
        tl, tr, to = tensor2d(lhs), tensor2d(rhs), tensor2d(out)
        ep = self._epilogue(alpha, bias, bias_axis, activation, rounding)
        st = self._lib.kapyb_matmul_host(self._h, C.byref(tl), C.byref(tr), C.byref(to),
                                         C.byref(ep), impl_way, self._stream(stream))
        if st != abi.OK:
            self._raise(st)
        return out

    def matmul_push(self, lhs, rhs_shard, peer_ptrs: Sequence[int], *, out_dtype, out_stride0: int,
                    col_begin: int, n_total: int, alpha: float = 1.0, bias=None,
                    activation: int = abi.ACT_NONE, rounding: int = abi.RN,
                    impl_way: int = abi.MMA_ANY, stream=None):
        """N-sharded matmul whose epilogue stores this rank's column block into
        every peer's full-size output (device pointers in `peer_ptrs`)."""
        tl, tr = tensor2d(lhs), tensor2d(rhs_shard)
        ep = self._epilogue(alpha, bias, 1, activation, rounding)
        arr = (C.c_void_p * len(peer_ptrs))(*[C.c_void_p(p) for p in peer_ptrs])
        st = self._lib.kapyb_matmul_push(self._h, C.byref(tl), C.byref(tr), arr, len(peer_ptrs),
                                         dtype_code(out_dtype), out_stride0, col_begin, n_total,
                                         C.byref(ep), impl_way, self._stream(stream))
        if st != abi.OK:
            self._raise(st)

    def gather_signal(self, peer_flag_ptrs: Sequence[int], my_rank: int, seq: int, stream=None):
        """Stores `seq` into word `my_rank` of every rank's flag array (device
        pointers), ordered after the work already on the stream."""
        arr = (C.c_void_p * len(peer_flag_ptrs))(*[C.c_void_p(p) for p in peer_flag_ptrs])
        st = self._lib.kapyb_gather_signal(self._h, arr, len(peer_flag_ptrs), int(my_rank),
                                           int(seq) & 0xFFFFFFFF, self._stream(stream))
        if st != abi.OK:
            self._raise(st)

    def gather_wait(self, my_flags_ptr: int, n_ranks: int, seq: int, limit_ms: int = 0,
                    stream=None):
        """Stream-ordered, bounded wait until every word of this rank's flag array
        has reached `seq`; a time-out surfaces in check()."""
        st = self._lib.kapyb_gather_wait(self._h, C.c_void_p(my_flags_ptr), int(n_ranks),
                                         int(seq) & 0xFFFFFFFF, int(limit_ms), self._stream(stream))
        if st != abi.OK:
            self._raise(st)

    def matmul_host_sharded(self, lhs_rows, m_total: int, row_begin: int, rhs, out, *,
                            peer_lhs_ptrs: Sequence[int], peer_flag_ptrs: Sequence[int], rank: int,
                            seq: int, wait_limit_ms: int = 0, alpha: float = 1.0, bias=None,
                            bias_axis: int = 1, activation: int = abi.ACT_NONE,
                            rounding: int = abi.RN, impl_way: int = abi.MMA_ANY, stream=None):
        """Host tensors in, host tensor out, on `len(peer_lhs_ptrs)` GPUs: this
        rank uploads rows [row_begin, row_begin + len(lhs_rows)) of lhs and its
        column block `rhs` of B, receives the other rows from its peers over
        NVLink, and computes out = lhs . rhs (see kapyb_matmul_host_sharded)."""
        for t in (lhs_rows, rhs, out):
            if t.is_cuda:
                raise ValueError("matmul_host_sharded takes host tensors")
        world = len(peer_lhs_ptrs)
        tl, tr, to = tensor2d(lhs_rows), tensor2d(rhs), tensor2d(out)
        ep = self._epilogue(alpha, bias, bias_axis, activation, rounding)
        pl = (C.c_void_p * world)(*[C.c_void_p(p) for p in peer_lhs_ptrs])
        pf = (C.c_void_p * world)(*[C.c_void_p(p) for p in peer_flag_ptrs])
        ctx = abi.ShardCtx(int(rank), world, pl, pf, int(seq) & 0xFFFFFFFF, int(wait_limit_ms))
        st = self._lib.kapyb_matmul_host_sharded(self._h, C.byref(tl), int(m_total), int(row_begin),
                                                 C.byref(tr), C.byref(to), C.byref(ep),
                                                 C.byref(ctx), impl_way, self._stream(stream))
        if st != abi.OK:
            self._raise(st)
        return out

    # ---------------------------------------------------- elementwise/reduce
    def elementwise(self, insts, inputs, out, paddings: Optional[Sequence[int]] = None,
                    stream=None, caches: Optional[Sequence[int]] = None, out_cache: int = 0):
        """Runs a recorded op list [(op,dtype,dst,a,b,c,imm,flags), ...].  `caches` /
        `out_cache`: abi.cache_hints(...) per input / for the output."""
        prog = (abi.Inst * max(1, len(insts)))()
        for i, t in enumerate(insts):
            prog[i] = abi.Inst(*t)
        tin = (abi.Tensor2d * max(1, len(inputs)))()
        for i, t in enumerate(inputs):
            tin[i] = tensor2d(t, paddings[i] if paddings else abi.PAD_ZERO,
                              caches[i] if caches else 0)
        to = tensor2d(out, cache=out_cache)
        st = self._lib.kapyb_elementwise(self._h, prog, len(insts), tin, len(inputs),
                                         C.byref(to), self._stream(stream))
        if st != abi.OK:
            self._raise(st)
        return out

    def reduce(self, src, axis: int, combiner: int = abi.RED_ADD, out=None, out_dtype=None,
               stream=None):
        """kapy.reduce along `axis` of a 2-D tensor; the reduced axis becomes 1."""
        torch = _torch()
        if out is None:
            shape = (1, src.shape[1]) if axis == 0 else (src.shape[0], 1)
            out = torch.empty(shape, device=src.device, dtype=out_dtype or src.dtype)
        ts, td = tensor2d(src), tensor2d(out)
        st = self._lib.kapyb_reduce(self._h, C.byref(ts), C.byref(td), int(axis), int(combiner),
                                    self._stream(stream))
        if st != abi.OK:
            self._raise(st)
        return out

    # ------------------------------------------- rows that pick their weights
    # These calls are often shorter than the host code in front of them, so that code
    # looks at each tensor once and builds nothing it does not pass on.
    def _launch_stream(self, stream):
        """(stream as an integer, context in which tensors the call allocates belong to it;
        None: the current stream, no context needed)."""
        if stream is None:
            return _current_stream(self.device), None
        torch = self._t
        if not hasattr(stream, "cuda_stream"):
            stream = torch.cuda.ExternalStream(int(stream), device=self.device)
        return stream.cuda_stream, torch.cuda.stream(stream)

    def _new(self, where, shape, dtype, zero=False):
        make = self._t.zeros if zero else self._t.empty
        if where is None:  # sizes one by one: a tuple of them costs torch 0.8 us more
            return make(*shape, dtype=dtype, device=self._torch_device)
        with where:
            return make(*shape, dtype=dtype, device=self._torch_device)

    def _fresh(self, where, rows, cols, dtype):
        """A new matrix and its descriptor."""
        t = self._new(where, (rows, cols), dtype)
        return t, _Tensor2d(t.data_ptr(), 0, rows, cols, max(1, cols), 1, _codes.get(dtype) or dtype_code(dtype))

    def _here(self, name, t):
        """The tensor's address, once it is known to be on the handle's GPU."""
        if t.get_device() != self.device:
            if not t.is_cuda:
                raise ValueError(f"{name} must be a CUDA tensor")
            raise ValueError(f"{name} is on {t.device}, the handle on cuda:{self.device}")
        return t.data_ptr()

    def _dense(self, name, t, dtype):
        """Address of a plain device array: right element type, contiguous, on the GPU."""
        if t.dtype is not dtype:
            raise ValueError(f"{name} must have element type {dtype}, not {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        return t.data_ptr() if t.get_device() == self.device else self._here(name, t)

    def _matrix(self, name, t):
        """Descriptor of a 2-D tensor on the handle's GPU."""
        if t.dim() != 2:
            raise ValueError("kapy tensors are rank 2")
        (rows, cols), (s0, s1) = t.shape, t.stride()
        if rows > _I32 or cols > _I32 or s0 > _I32 or s1 > _I32:
            raise ValueError("sizes and strides must fit i32")
        at = t.data_ptr() if t.get_device() == self.device else self._here(name, t)
        return _Tensor2d(at, 0, rows, cols, s0, s1, _codes.get(t.dtype) or dtype_code(t.dtype))

    def _stack(self, name, t):
        """Descriptor of the first matrix of [groups, rows, columns] and the group stride."""
        if t.dim() != 3:
            raise ValueError(f"{name} must be [groups, rows, columns]")
        (_, rows, cols), (stride, s0, s1) = t.shape, t.stride()
        if rows > _I32 or cols > _I32 or s0 > _I32 or s1 > _I32:
            raise ValueError("sizes and strides must fit i32")
        at = t.data_ptr() if t.get_device() == self.device else self._here(name, t)
        return _Tensor2d(at, 0, rows, cols, s0, s1, _codes.get(t.dtype) or dtype_code(t.dtype)), stride

    def route(self, logits, top_k: int, *, bias=None, score: int = abi.SCORE_SOFTMAX,
              groups: int = 1, top_groups: Optional[int] = None, group_best: int = 1,
              renormalize: bool = True, scale: float = 1.0, weights=None, experts=None,
              stream=None):
        """Routing of rows to experts (kapyb_route): (weights f32 [T, k], experts int32
        [T, k]) of logits [T, E]; the bias (f32 [E]) takes part in the choice only."""
        torch = self._t
        tl = self._matrix("logits", logits)
        shape = (tl.size0, int(top_k))
        at_bias = None
        if bias is not None:
            if bias.shape != (tl.size1,):
                raise ValueError("bias must have one value per expert")
            at_bias = self._dense("bias", bias, torch.float32)
        r = abi.Routing(int(score), shape[1], int(groups),
                        int(groups if top_groups is None else top_groups), int(group_best),
                        1 if renormalize else 0, float(scale))
        s, where = self._launch_stream(stream)
        held = (shape[0], max(0, shape[1]))  # a refused top_k is refused by the call itself
        if weights is None:
            weights = self._new(where, held, torch.float32)
            at_weights = weights.data_ptr()
        elif weights.shape != shape:
            raise ValueError(f"weights must have shape {shape}")
        else:
            at_weights = self._dense("weights", weights, torch.float32)
        if experts is None:
            experts = self._new(where, held, torch.int32)
            at_experts = experts.data_ptr()
        elif experts.shape != shape:
            raise ValueError(f"experts must have shape {shape}")
        else:
            at_experts = self._dense("experts", experts, torch.int32)
        st = self._lib.kapyb_route(self._h, tl, at_bias, r, at_weights, at_experts, s)
        if st != abi.OK:
            self._raise(st)
        return weights, experts

    def route_backward(self, logits, experts, grad_weights, *, score: int = abi.SCORE_SOFTMAX,
                       renormalize: bool = True, scale: float = 1.0, out=None, stream=None):
        """Gradient of the logits (kapyb_route_backward) from the gradient of route's
        weights; `experts`, score, renormalize and scale as in the forward call."""
        torch = self._t
        tl = self._matrix("logits", logits)
        if experts.dim() != 2 or experts.shape[0] != tl.size0 or \
                grad_weights.shape != experts.shape:
            raise ValueError("experts and grad_weights must be [rows of logits, k]")
        r = abi.Routing(int(score), experts.shape[1], 1, 1, 1, 1 if renormalize else 0, float(scale))
        s, where = self._launch_stream(stream)
        if out is None:
            out = self._new(where, logits.shape, logits.dtype)
        st = self._lib.kapyb_route_backward(
            self._h, tl, r, self._dense("experts", experts, torch.int32),
            self._dense("grad_weights", grad_weights, torch.float32), self._matrix("out", out), s)
        if st != abi.OK:
            self._raise(st)
        return out

    def plan_rows(self, index, groups: int, *, order=None, offsets=None, slots=None, stream=None):
        """Stable counting sort of an int32 index (any shape) into groups
        (kapyb_plan_rows): (order [n], offsets [groups + 1], slots of index's shape)."""
        torch = self._t
        n, groups = index.numel(), int(groups)
        s, where = self._launch_stream(stream)
        def place(name, t, shape, count):
            if t is None:
                t = self._new(where, shape, torch.int32)
                return t, t.data_ptr()
            if t.numel() != count:
                raise ValueError(f"{name} must have {count} elements")
            return t, self._dense(name, t, torch.int32)

        order, at_order = place("order", order, (n,), n)
        offsets, at_offsets = place("offsets", offsets, (max(0, groups) + 1,), groups + 1)
        slots, at_slots = place("slots", slots, index.shape or (1,), n)
        st = self._lib.kapyb_plan_rows(self._h, self._dense("index", index, torch.int32), n, groups,
                                       at_order, at_offsets, at_slots, s)
        if st != abi.OK:
            self._raise(st)
        return order, offsets, slots

    def _plan(self, offsets, order, fan, groups, rows):
        """Addresses of a plan's offsets and order."""
        torch = self._t
        if offsets.numel() != groups + 1:
            raise ValueError(f"offsets must have {groups + 1} elements")
        at = self._dense("offsets", offsets, torch.int32)
        if order is None:
            return at, None
        if order.numel() != rows:
            raise ValueError(f"order must have {rows} elements")
        if int(fan) < 1:
            raise ValueError("fan must be at least 1")
        return at, self._dense("order", order, torch.int32)

    def matmul_grouped(self, lhs, rhs, offsets, out=None, *, order=None, fan: int = 1,
                       alpha: float = 1.0, bias=None, activation: int = abi.ACT_NONE,
                       gated: bool = False, rounding: int = abi.RN, out_dtype=None, stream=None):
        """out[p] = epilogue(lhs[row] . rhs[g]) for every planned position p of group g
        (kapyb_matmul_grouped): row = order[p] // fan, or p without an order.  rhs is
        [groups, K, N]; gated: [groups, K, 2 N], gate columns then up columns, out =
        activation(gate) * up.  bias: [groups, columns of rhs]."""
        tl = self._matrix("lhs", lhs)
        tr, group_stride = self._stack("rhs", rhs)
        groups = rhs.shape[0]
        rows = order.numel() if order is not None else tl.size0
        at_offsets, at_order = self._plan(offsets, order, fan, groups, rows)
        if bias is not None:
            if bias.shape != (groups, tr.size1):
                raise ValueError("bias must be [groups, columns of rhs]")
            self._here("bias", bias)
        s, where = self._launch_stream(stream)
        if out is None:
            out, to = self._fresh(where, rows, tr.size1 // 2 if gated else tr.size1, out_dtype or lhs.dtype)
        elif out.shape[0] != rows:
            raise ValueError(f"out must have {rows} rows")
        else:
            to = self._matrix("out", out)
        ep = None  # nothing to apply: the call's default
        if bias is not None or activation or alpha != 1.0 or rounding != abi.RN:
            ep = self._epilogue(alpha, bias, 1, activation, rounding)
        st = self._lib.kapyb_matmul_grouped(self._h, tl, tr, groups, group_stride, at_offsets,
                                            at_order, int(fan), to, ep, 1 if gated else 0, s)
        if st != abi.OK:
            self._raise(st)
        return out

    def matmul_grouped_grad(self, lhs, grad, offsets, out=None, *, order=None, fan: int = 1,
                            alpha: float = 1.0, rounding: int = abi.RN, out_dtype=None,
                            stream=None):
        """Gradient of matmul_grouped's weights (kapyb_matmul_grouped_grad): [groups, K, N]
        from lhs, the gradient of the products [positions, N] and the plan they ran on."""
        tl, tg = self._matrix("lhs", lhs), self._matrix("grad", grad)
        groups = offsets.numel() - 1
        at_offsets, at_order = self._plan(offsets, order, fan, groups, tg.size0)
        s, where = self._launch_stream(stream)
        if out is None:
            out = self._new(where, (groups, tl.size1, tg.size1), out_dtype or lhs.dtype)
        elif out.shape[0] != groups:
            raise ValueError(f"out must have {groups} groups")
        to, group_stride = self._stack("out", out)
        st = self._lib.kapyb_matmul_grouped_grad(self._h, tl, tg, groups, at_offsets, at_order,
                                                 int(fan), to, group_stride, float(alpha),
                                                 int(rounding), s)
        if st != abi.OK:
            self._raise(st)
        return out

    def combine_rows(self, rows, slots, out=None, *, weights=None, out_dtype=None, stream=None):
        """out[t] = sum_j weights[t, j] * rows[slots[t, j]] (kapyb_combine_rows)."""
        torch = self._t
        tr = self._matrix("rows", rows)
        if slots.dim() != 2 or (weights is not None and weights.shape != slots.shape):
            raise ValueError("slots and weights must be [tokens, k]")
        tokens, k = slots.shape
        s, where = self._launch_stream(stream)
        if out is None:
            out, to = self._fresh(where, tokens, tr.size1, out_dtype or rows.dtype)
        elif out.shape[0] != tokens:
            raise ValueError("out must have a row per token")
        else:
            to = self._matrix("out", out)
        st = self._lib.kapyb_combine_rows(
            self._h, tr, self._dense("slots", slots, torch.int32), k,
            None if weights is None else self._dense("weights", weights, torch.float32), to, s)
        if st != abi.OK:
            self._raise(st)
        return out

    def combine_rows_backward(self, rows, slots, grad_out, *, weights=None, grad_rows=None,
                              grad_weights=None, stream=None):
        """Gradients of combine_rows (kapyb_combine_rows_backward): (grad_rows,
        grad_weights); the latter is None for a sum without weights.  A given grad_rows
        keeps the rows no slot names; an allocated one starts as zeros."""
        torch = self._t
        tr, tg = self._matrix("rows", rows), self._matrix("grad_out", grad_out)
        if slots.dim() != 2 or tg.size0 != slots.shape[0] or \
                any(t is not None and t.shape != slots.shape for t in (weights, grad_weights)):
            raise ValueError("slots, weights and grad_weights must be [rows of grad_out, k]")
        s, where = self._launch_stream(stream)
        if grad_rows is None:
            grad_rows = self._new(where, rows.shape, rows.dtype, zero=True)
        if grad_weights is None and weights is not None:
            grad_weights = self._new(where, slots.shape, torch.float32)
        st = self._lib.kapyb_combine_rows_backward(
            self._h, tr, self._dense("slots", slots, torch.int32), slots.shape[1],
            None if weights is None else self._dense("weights", weights, torch.float32), tg,
            self._matrix("grad_rows", grad_rows),
            None if grad_weights is None else self._dense("grad_weights", grad_weights, torch.float32),
            s)
        if st != abi.OK:
            self._raise(st)
        return grad_rows, grad_weights

    def matmul_adapters(self, lhs, rhs, down, up, index, out=None, *, scale=None,
                        alpha: float = 1.0, bias=None, bias_axis: int = 1,
                        activation: int = abi.ACT_NONE, rounding: int = abi.RN, out_dtype=None,
                        stream=None):
        """lhs . rhs with every row's low-rank adapter beside it (kapyb_matmul_adapters):
        row t adds scale[i] * (lhs[t] . down[i]) . up[i], i = index[t]; an index outside
        the adapters adds nothing.  down [groups, K, rank], up [groups, rank, N]."""
        torch = self._t
        tl, tr = self._matrix("lhs", lhs), self._matrix("rhs", rhs)
        td, down_stride = self._stack("down", down)
        tu, up_stride = self._stack("up", up)
        groups = down.shape[0]
        if up.shape[0] != groups or (scale is not None and scale.numel() != groups):
            raise ValueError("down, up and scale must have as many adapters")
        if index.numel() != tl.size0:
            raise ValueError("index must have an element per row of lhs")
        if bias is not None:
            if bias.numel() != (tr.size1 if bias_axis == 1 else tl.size0):
                raise ValueError("bias must have a value per column (bias_axis 1) or row (0)")
            self._here("bias", bias)
        s, where = self._launch_stream(stream)
        nbytes = self._lib.kapyb_matmul_adapters_scratch(tl.size0, groups, td.size1)
        scratch = self._new(where, (nbytes,), torch.uint8)
        if out is None:
            out, to = self._fresh(where, tl.size0, tr.size1, out_dtype or lhs.dtype)
        else:
            to = self._matrix("out", out)
        ep = None  # nothing to apply: the call's default
        if bias is not None or activation or alpha != 1.0 or rounding != abi.RN or bias_axis != 1:
            ep = self._epilogue(alpha, bias, bias_axis, activation, rounding)
        st = self._lib.kapyb_matmul_adapters(
            self._h, tl, tr, groups, td, down_stride, tu, up_stride,
            self._dense("index", index, torch.int32),
            None if scale is None else self._dense("scale", scale, torch.float32),
            to, ep, scratch.data_ptr(), nbytes, s)
        if st != abi.OK:
            self._raise(st)
        return out


def shard_range(total: int, parts: int, rank: int, align: int = 1):
    """[begin, end) of `total` units owned by `rank` (blocks of `align`)."""
    lib = abi.load()
    b, e = C.c_int64(), C.c_int64()
    st = lib.kapyb_shard_range(total, parts, rank, align, C.byref(b), C.byref(e))
    if st != abi.OK:
        raise ValueError("bad shard arguments")
    return int(b.value), int(e.value)
