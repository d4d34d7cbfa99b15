"""sffft_b200: B200 (sm_100a) fused causal long convolution.

    y[b, h, n] = sum_{m <= n} u[b, h, m] * k[h, n - m],   n < L

Python mirror of the C ABI in ``include/sffft.h`` (itself the drop-in for the operator surface of
sfFFT's ``src/sffft.cu`` and ``src/selection.h``).  Device buffers are torch CUDA tensors (or raw
device pointers); every native call raises :class:`SffftError` on a non-zero status.  There is no CPU
fallback: if ``lib/libsffft.so`` is missing or the device is not a B200, calls fail.
"""
from __future__ import annotations

import ctypes
import functools
import math
import os
import struct
from dataclasses import dataclass
from typing import Optional, Sequence

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libsffft.so")
TORCH_LIB_PATH = os.path.join(_HERE, "lib", "libsffft_torch.so")   # the PyTorch operators (torch_ops)
EMU_PATH = os.path.join(_HERE, "lib", "libsffft_emu.so")
CLI_PATH = os.path.join(_HERE, "bin", "sffft")

(OK, ERR_INVALID_ARGUMENT, ERR_UNSUPPORTED, ERR_CUDA, ERR_DEVICE, ERR_TIMEOUT, ERR_NO_MATCH, ERR_ALLOC,
 ERR_SCRATCH_LIMIT, ERR_WORKSPACE) = range(10)
IO = {"fp32": 0, "bf16": 1}
ACC = {"fp32": 0, "fp16": 1}
KERNEL = {"legacy": 0, "cached": 1}
FILTER = {"causal": 0, "two_sided": 1, "circular": 2}
GATE = {"none": 0, "full": 1, "channel": 2}
ACT = {"none": 0, "silu": 1, "sigmoid": 2}

_lib = None
_emu = None


class SffftError(RuntimeError):
    def __init__(self, status: int, what: str):
        self.status = status
        super().__init__(f"{what}: {status_string(status) if _lib else status} (status {status})")


class PlanInfo(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int) for n in (
        "L", "N", "stages", "R0", "R1", "R2", "pairs_per_cta", "warps", "threads", "smem_bytes",
        "tmem_cols", "occupancy", "io", "acc", "kernel_mode", "device", "blocks")] + [("config", ctypes.c_char * 96)]


class LinearAttentionDesc(ctypes.Structure):
    """sffft_linear_attention_t"""
    _fields_ = ([(n, ctypes.c_int) for n in ("B", "H", "Hkv", "L", "D", "Dv", "io", "device")] + [("scale", ctypes.c_float)]
                + [(n, ctypes.c_longlong * 3) for n in ("q_stride", "k_stride", "v_stride", "y_stride")])


class LinearAttentionGrads(ctypes.Structure):
    """sffft_linear_attention_grads_t"""
    _fields_ = [(n, ctypes.c_longlong * 3) for n in ("dy_stride", "dq_stride", "dk_stride", "dv_stride")]


class LinearAttentionStepDesc(ctypes.Structure):
    """sffft_linear_attention_step_t"""
    _fields_ = ([(n, ctypes.c_int) for n in ("B", "H", "Hkv", "D", "Dv", "pool", "io", "device")] + [("scale", ctypes.c_float)]
                + [(n, ctypes.c_longlong * 2) for n in ("q_stride", "k_stride", "v_stride", "y_stride")]
                + [("state_stride", ctypes.c_longlong)])


class BlockNormDesc(ctypes.Structure):
    """sffft_block_norm_t"""
    _fields_ = ([("rows", ctypes.c_longlong)]
                + [(n, ctypes.c_int) for n in ("channels", "inner", "groups", "io", "res_io", "weight_io", "gate", "act")]
                + [("scale", ctypes.c_float), ("eps", ctypes.c_float), ("device", ctypes.c_int)]
                + [(n, ctypes.c_longlong) for n in ("x_stride", "y_stride", "gate_stride")])


class _Candidate(ctypes.Structure):
    _fields_ = [("method", ctypes.c_char_p), ("io", ctypes.c_char_p), ("config", ctypes.c_char_p),
                ("ms", ctypes.c_double), ("rel_err", ctypes.c_double)]


def _declare(lib):
    P, I, V, D = ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_double
    sig = {
        "sffft_plan_create": (I, [ctypes.POINTER(P), I, I, I, ctypes.c_char_p, I, I]),
        "sffft_plan_destroy": (I, [P]),
        "sffft_plan_info": (I, [P, ctypes.POINTER(PlanInfo)]),
        "sffft_filter_spectrum": (I, [P, V, I, I, V, V]),
        "sffft_filter_spectrum_ex": (I, [P, V, I, I, I, V, V]),
        "sffft_fft_workspace_bytes": (I, [P, I, ctypes.POINTER(ctypes.c_size_t)]),
        "sffft_rfft": (I, [P, V, I, I, V, V, V]),
        "sffft_irfft": (I, [P, V, I, V, V, V]),
        "sffft_conv": (I, [P, V, V, V, I, I, V]),
        "sffft_conv_workspace_bytes": (I, [P, I, I, ctypes.POINTER(ctypes.c_size_t)]),
        "sffft_conv_ws": (I, [P, V, V, V, I, I, V, ctypes.c_size_t, V]),
        "sffft_plan_set_workspace": (I, [P, V, ctypes.c_size_t]),
        "sffft_plan_check": (I, [P]),
        "sffft_catalog_count": (I, []),
        "sffft_catalog_entry": (I, [I, ctypes.POINTER(I), ctypes.c_char_p, I]),
        "sffft_default_config": (I, [I, ctypes.c_char_p, I]),
        "sffft_select_candidate": (I, [ctypes.POINTER(_Candidate), I, D, ctypes.c_char_p]),
        "sffft_relative_l2": (D, [D, D]),
        "sffft_shard_range": (I, [I, I, I, ctypes.POINTER(I), ctypes.POINTER(I)]),
        "sffft_status_string": (ctypes.c_char_p, [I]),
        "sffft_last_cuda_error": (I, []),
        "sffft_baseline_create": (I, [ctypes.POINTER(P), I, I, I, V, I]),
        "sffft_baseline_run": (I, [P, V, V, I, V]),
        "sffft_baseline_destroy": (I, [P]),
        "sffft_debug_umma_probe": (I, [I, I, I, I, I, I, V, V, V]),
        "sffft_debug_wait_timeout": (I, [I]),
        "sffft_debug_linear_attention": (I, [I, I]),
        "sffft_debug_conv_timeout": (I, [P, V, V, V, I, I, I, V]),
        "sffft_conv_noalloc": (I, [I, I, I, V, V, I, V, I, I, V, I]),
        "sffft_pipe_create": (I, [ctypes.POINTER(P), P, I, I, I]),
        "sffft_conv_host": (I, [P, V, V, V, V]),
        "sffft_pipe_destroy": (I, [P]),
        "sffft_conv_multi": (I, [ctypes.POINTER(P), I, ctypes.POINTER(V), ctypes.POINTER(V), ctypes.POINTER(V), I, I,
                                 ctypes.POINTER(V)]),
        "sffft_multi_pipe_create": (I, [ctypes.POINTER(P), ctypes.POINTER(P), I, I, I, I]),
        "sffft_conv_host_multi": (I, [P, V, ctypes.POINTER(V), V]),
        "sffft_multi_pipe_destroy": (I, [P]),
        "sffft_linear_attention_workspace_bytes": (I, [V, I, ctypes.POINTER(ctypes.c_size_t)]),
        "sffft_linear_attention": (I, [V] * 10 + [ctypes.c_size_t, V]),
        "sffft_linear_attention_backward": (I, [V] * 15 + [ctypes.c_size_t, V]),
        "sffft_linear_attention_check": (I, [I]),
        "sffft_linear_attention_step": (I, [V] * 9),
        "sffft_block_norm": (I, [V] * 11),
        "sffft_block_norm_workspace_bytes": (I, [V, ctypes.POINTER(ctypes.c_size_t)]),
        "sffft_block_norm_backward": (I, [V] * 16 + [ctypes.c_size_t, V]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype, fn.argtypes = res, args
    return lib


def lib():
    """The native library (loaded once).  Raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"native library missing: {LIB_PATH} (run `make -C sffft_b200`)")
        _lib = _declare(ctypes.CDLL(LIB_PATH))
    return _lib


def _check(status: int, what: str):
    if status != OK:
        raise SffftError(status, what)


def status_string(status: int) -> str:
    return lib().sffft_status_string(status).decode()


def _ptr(x) -> Optional[int]:
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return x.data_ptr()


def _stream(stream) -> Optional[int]:
    if stream is None:
        return None
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def catalog() -> list[tuple[int, str]]:
    """(L, name) of every compiled plan."""
    L = lib()
    out = []
    buf = ctypes.create_string_buffer(96)
    for i in range(L.sffft_catalog_count()):
        n = ctypes.c_int()
        _check(L.sffft_catalog_entry(i, ctypes.byref(n), buf, 96), "catalog")
        out.append((n.value, buf.value.decode()))
    return out


def default_config(L: int) -> str:
    buf = ctypes.create_string_buffer(96)
    _check(lib().sffft_default_config(L, buf, 96), f"default config for L={L}")
    return buf.value.decode()


def relative_l2(squared_error: float, squared_reference: float) -> float:
    """relative_l2 of src/selection.h:26-29."""
    return lib().sffft_relative_l2(squared_error, squared_reference)


@dataclass
class Candidate:
    """Candidate of src/selection.h:8-11."""
    method: str
    io: str
    config: str
    ms: float
    rel_err: float


def select_candidate(candidates: Sequence[Candidate], max_error: float, io: str) -> Optional[int]:
    """Index of select_candidate's choice (src/selection.h:13-24), or None."""
    arr = (_Candidate * max(1, len(candidates)))()
    keep = []
    for i, c in enumerate(candidates):
        fields = [c.method.encode(), c.io.encode(), c.config.encode()]
        keep.append(fields)
        arr[i] = _Candidate(fields[0], fields[1], fields[2], float(c.ms), float(c.rel_err))
    idx = lib().sffft_select_candidate(arr, len(candidates), float(max_error), io.encode())
    return None if idx < 0 else idx


def shard_range(H: int, shards: int, shard: int) -> tuple[int, int]:
    """Contiguous channel range [h0, h1) owned by `shard` of `shards`."""
    h0, h1 = ctypes.c_int(), ctypes.c_int()
    _check(lib().sffft_shard_range(H, shards, shard, ctypes.byref(h0), ctypes.byref(h1)), "shard_range")
    return h0.value, h1.value


class Plan:
    """A compiled fused-convolution plan for one length, I/O type, accumulation mode and device.

    Mirrors the reference's fftconv<Plan<R0,R1,R2>,W,TIO,TAcc,CACHED> choice (src/sffft.cu:243-245)."""

    def __init__(self, L: int, io: str = "fp32", acc: str = "fp32", config: Optional[str] = None,
                 kernel: str = "cached", device: int = 0):
        self._h = ctypes.c_void_p()
        cfg = config.encode() if config else None
        _check(lib().sffft_plan_create(ctypes.byref(self._h), L, IO[io], ACC[acc], cfg, KERNEL[kernel], device),
               f"plan_create(L={L}, io={io}, acc={acc}, config={config})")
        self.L, self.io, self.acc, self.kernel, self.device = L, io, acc, kernel, device
        inf = PlanInfo()
        _check(lib().sffft_plan_info(self._h, ctypes.byref(inf)), "plan_info")
        self.info = {f: getattr(inf, f) for f, _ in PlanInfo._fields_ if f != "config"}
        self.info["config"] = inf.config.decode()
        self.config = self.info["config"]
        self.N = inf.N
        self.blocks = inf.blocks
        # digits of the length-N transform; a composite plan's last digit spans its blocks
        self.radices = [r for r in (inf.R0, inf.R1, inf.R2) if r > 1]
        self.radices[-1] *= self.blocks
        self._ws = None   # composite plans: the workspace of conv (a device byte tensor, grown on demand)

    def filter_spectrum(self, k, Kf=None, stream=None, layout="causal"):
        """Kf [H][N] complex fp32 (as float32 [H, N, 2]) in digit order from the filter k.

        layout "causal": k [H][L], conv gives y[n] = sum_{m<=n} u[m] k[n-m] (the reference's form);
        "two_sided": k [H][2L-1], y[n] = sum_{m<L} u[m] k[L-1+n-m] (k[:, L-1] is lag 0);
        "circular": k [H][L], y[n] = sum_{m<L} u[m] k[(n-m) mod L]."""
        import torch
        if layout not in FILTER:
            raise ValueError(f"layout must be one of {sorted(FILTER)}")
        width = 2 * self.L - 1 if layout == "two_sided" else self.L
        if k.dim() != 2 or k.shape[1] != width or k.dtype not in (torch.float32, torch.bfloat16) or not k.is_contiguous():
            raise ValueError(f"k must be a contiguous [H][{width}] float32 or bfloat16 tensor for layout {layout!r}")
        H = k.shape[0]
        if Kf is None:
            Kf = torch.empty((H, self.N, 2), dtype=torch.float32, device=k.device)
        kd = IO["bf16"] if k.dtype == torch.bfloat16 else IO["fp32"]
        _check(lib().sffft_filter_spectrum_ex(self._h, _ptr(k), kd, FILTER[layout], H, _ptr(Kf), _stream(stream)),
               "filter_spectrum")
        return Kf

    def _fft_work(self, rows, work, device):
        import torch
        need = ctypes.c_size_t()
        _check(lib().sffft_fft_workspace_bytes(self._h, rows, ctypes.byref(need)), "fft_workspace_bytes")
        if work is None:
            return torch.empty(need.value // 4, dtype=torch.float32, device=device)
        if work.numel() * work.element_size() < need.value:
            raise ValueError(f"workspace of {need.value} bytes needed")
        return work

    def rfft(self, x, X=None, work=None, stream=None):
        """X [..., N/2+1] complex64 = the length-N real DFT of x [..., N] (fp32 or bf16), numpy.fft.rfft's
        definition; N = 2L is the plan's transform length."""
        import torch
        if x.shape[-1] != self.N or x.dtype not in (torch.float32, torch.bfloat16) or not x.is_contiguous():
            raise ValueError(f"x must be a contiguous [..., {self.N}] float32 or bfloat16 tensor")
        rows = x.numel() // self.N
        if X is None:
            X = torch.empty(tuple(x.shape[:-1]) + (self.N // 2 + 1,), dtype=torch.complex64, device=x.device)
        work = self._fft_work(rows, work, x.device)
        kd = IO["bf16"] if x.dtype == torch.bfloat16 else IO["fp32"]
        _check(lib().sffft_rfft(self._h, _ptr(x), kd, rows, _ptr(X), _ptr(work), _stream(stream)), "rfft")
        return X

    def irfft(self, X, x=None, work=None, stream=None):
        """x [..., N] fp32 = the inverse of rfft for the half spectrum X [..., N/2+1] complex64
        (numpy.fft.irfft's definition, 1/N included)."""
        import torch
        if X.shape[-1] != self.N // 2 + 1 or X.dtype != torch.complex64 or not X.is_contiguous():
            raise ValueError(f"X must be a contiguous [..., {self.N // 2 + 1}] complex64 tensor")
        rows = X.numel() // (self.N // 2 + 1)
        if x is None:
            x = torch.empty(tuple(X.shape[:-1]) + (self.N,), dtype=torch.float32, device=X.device)
        work = self._fft_work(rows, work, X.device)
        _check(lib().sffft_irfft(self._h, _ptr(X), rows, _ptr(x), _ptr(work), _stream(stream)), "irfft")
        return x

    def workspace_bytes(self, B: int, H: int) -> int:
        """Device workspace of a B x H convolution (sffft_conv_workspace_bytes): 0 for single-pass plans."""
        need = ctypes.c_size_t()
        _check(lib().sffft_conv_workspace_bytes(self._h, B, H, ctypes.byref(need)), "conv_workspace_bytes")
        return need.value

    def _work(self, B, H, work):
        need = self.workspace_bytes(B, H)
        if need == 0:
            return None, 0
        if work is not None:
            nbytes = work.numel() * work.element_size()
            if nbytes < need:
                raise ValueError(f"workspace of {need} bytes needed, got {nbytes}")
            return work.data_ptr(), nbytes
        import torch
        if self._ws is None or self._ws.numel() < need:
            self._ws = None
            self._ws = torch.empty(need, dtype=torch.uint8, device=torch.device("cuda", self.device))
        return self._ws.data_ptr(), self._ws.numel()

    def conv(self, u, Kf, y=None, stream=None, work=None):
        """y = causal_conv(u, k) for u [B][H][L] with the spectrum Kf of k.  Composite plans use `work` (a device
        tensor of at least workspace_bytes(B, H) bytes) or a workspace the plan keeps for its calls."""
        import torch
        B, H, L = u.shape
        if L != self.L:
            raise ValueError(f"plan is for L={self.L}, got {L}")
        if y is None:
            y = torch.empty_like(u)
        wp, wn = self._work(B, H, work)
        _check(lib().sffft_conv_ws(self._h, _ptr(u), _ptr(Kf), _ptr(y), B, H, wp, wn, _stream(stream)), "conv")
        return y

    def conv_ptr(self, u_ptr: int, Kf_ptr: int, y_ptr: int, B: int, H: int, stream=None) -> int:
        """Raw-pointer form; returns the status instead of raising (for tight timing loops)."""
        wp, wn = self._work(B, H, None) if self.blocks > 1 else (None, 0)
        return lib().sffft_conv_ws(self._h, u_ptr, Kf_ptr, y_ptr, B, H, wp, wn, _stream(stream))

    def check(self):
        """Synchronise and raise if a kernel reported a device-side error."""
        _check(lib().sffft_plan_check(self._h), "device status")

    def close(self):
        if self._h:
            lib().sffft_plan_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class HostPipe:
    """Convolution of a batch held in host memory (sffft_pipe_create / sffft_conv_host): chunks of batch-row
    pairs are uploaded, convolved and downloaded on three streams so the copies and the kernels overlap."""

    def __init__(self, plan: "Plan", B: int, H: int, chunks: int = 0):
        self._h = ctypes.c_void_p()
        _check(lib().sffft_pipe_create(ctypes.byref(self._h), plan._h, B, H, chunks), "pipe_create")
        self.plan, self.B, self.H = plan, B, H

    def conv(self, u_host, Kf, y_host, stream=None):
        """y_host = causal_conv(u_host, k) for host tensors u_host, y_host [B][H][L] and the device spectrum Kf."""
        if tuple(u_host.shape) != (self.B, self.H, self.plan.L) or tuple(y_host.shape) != tuple(u_host.shape):
            raise ValueError("u_host / y_host must be [B][H][L] of the pipe's batch")
        _check(lib().sffft_conv_host(self._h, _ptr(u_host), _ptr(Kf), _ptr(y_host), _stream(stream)), "conv_host")
        return y_host

    def close(self):
        if self._h:
            lib().sffft_pipe_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _ptr_array(items):
    arr = (ctypes.c_void_p * len(items))()
    for i, x in enumerate(items):
        arr[i] = _ptr(x)
    return arr


def conv_multi(plans: Sequence["Plan"], us, Kfs, ys, B: int, H: int, streams=None):
    """Channel-sharded convolution of device-resident shards (sffft_conv_multi): shard g = channels
    shard_range(H, len(plans), g) on plans[g]'s device, u[g]/y[g] [B][h1-h0][L], Kf[g] [h1-h0][N]."""
    G = len(plans)
    hs = (ctypes.c_void_p * G)(*[p._h.value for p in plans])
    st = _ptr_array([_stream(s) for s in streams]) if streams is not None else None
    _check(lib().sffft_conv_multi(hs, G, _ptr_array(us), _ptr_array(Kfs), _ptr_array(ys), B, H, st), "conv_multi")
    return ys


class HostPipeMulti:
    """One [B][H][L] host batch convolved by several devices (sffft_multi_pipe_create / sffft_conv_host_multi):
    device g takes channels shard_range(H, len(plans), g) through a host pipe of its own; conv() returns when
    every device is done."""

    def __init__(self, plans: Sequence["Plan"], B: int, H: int, chunks: int = 0):
        self._h = ctypes.c_void_p()
        G = len(plans)
        hs = (ctypes.c_void_p * G)(*[p._h.value for p in plans])
        _check(lib().sffft_multi_pipe_create(ctypes.byref(self._h), hs, G, B, H, chunks), "multi_pipe_create")
        self.plans, self.B, self.H = list(plans), B, H

    def conv(self, u_host, Kfs, y_host):
        if tuple(u_host.shape) != (self.B, self.H, self.plans[0].L) or tuple(y_host.shape) != tuple(u_host.shape):
            raise ValueError("u_host / y_host must be [B][H][L] of the pipe's batch")
        _check(lib().sffft_conv_host_multi(self._h, _ptr(u_host), _ptr_array(Kfs), _ptr(y_host)), "conv_host_multi")
        return y_host

    def close(self):
        if self._h:
            lib().sffft_multi_pipe_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Baseline:
    """cuFFT pipeline (pad -> R2C -> x spectrum -> C2R -> slice) of src/sffft.cu:289-305,365-371."""

    def __init__(self, L: int, B: int, H: int, k, device: int = 0):
        self._h = ctypes.c_void_p()
        _check(lib().sffft_baseline_create(ctypes.byref(self._h), L, B, H, _ptr(k), device), "baseline_create")

    def run(self, u, y=None, full: bool = True, stream=None):
        _check(lib().sffft_baseline_run(self._h, _ptr(u), _ptr(y), 1 if full else 0, _stream(stream)), "baseline_run")
        return y

    def close(self):
        if self._h:
            lib().sffft_baseline_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def umma_probe(a_kind: int, a_slice: int, b_pitch: int, b_slice: int, A, Bm, acc16: bool = False):
    """One tcgen05.mma through the kernel's layout writers (debug).  A: uint16 [128,16], Bm: uint16 [n,16];
    returns uint32 [128, n] raw TMEM words."""
    import numpy as np
    A = np.ascontiguousarray(A, dtype=np.uint16)
    Bm = np.ascontiguousarray(Bm, dtype=np.uint16)
    n = Bm.shape[0]
    D = np.zeros((128, n), dtype=np.uint32)
    _check(lib().sffft_debug_umma_probe(a_kind, a_slice, b_pitch, b_slice, n, 1 if acc16 else 0,
                                        A.ctypes.data, Bm.ctypes.data, D.ctypes.data), "umma_probe")
    return D


def _emu_lib():
    global _emu
    if _emu is None:
        if not os.path.exists(EMU_PATH):
            raise RuntimeError(f"emulator library missing: {EMU_PATH}")
        _emu = ctypes.CDLL(EMU_PATH)
        _emu.sffft_emu_conv.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_int, ctypes.c_void_p,
                                        ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int]
        _emu.sffft_emu_conv_composite.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_int, ctypes.c_int,
                                                  ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int,
                                                  ctypes.c_int]
    return _emu


def emu_conv_composite(config: str, P: int, u, Kf, io: str = "fp32", acc: str = "fp32"):
    """CPU emulation of the composite plan "<P>x[<config>]" (row energies, forward and inverse launches of the
    partitioned convolution); Kf: the P filter-segment spectra [P][H][N] (float32 pairs).  Test infrastructure."""
    import numpy as np
    B, H, L = u.shape
    u = np.ascontiguousarray(u)
    Kf = np.ascontiguousarray(Kf, dtype=np.float32)
    y = np.zeros_like(u)
    rc = _emu_lib().sffft_emu_conv_composite(config.encode(), P, IO[io], ACC[acc], u.ctypes.data, Kf.ctypes.data,
                                             y.ctypes.data, B, H)
    if rc == 3:
        raise RuntimeError(f"emulated kernel accessed memory out of range ({P}x[{config}])")
    if rc:
        raise ValueError(f"no partitioned-convolution kernels for {config}")
    return y


def emu_conv(config: str, u, Kf, io: str = "fp32", acc: str = "fp32"):
    """CPU emulation of the fused kernel (same stage code, emulated tcgen05); numpy in and out.
    Test infrastructure for checking layouts without a GPU."""
    import numpy as np
    B, H, L = u.shape
    u = np.ascontiguousarray(u)
    Kf = np.ascontiguousarray(Kf, dtype=np.float32)
    y = np.zeros_like(u)
    rc = _emu_lib().sffft_emu_conv(config.encode(), IO[io], ACC[acc], u.ctypes.data, Kf.ctypes.data, y.ctypes.data, B, H)
    if rc == 3:
        raise RuntimeError(f"emulated kernel accessed shared memory or TMEM out of range ({config})")
    if rc:
        raise ValueError(f"unknown config {config}")
    return y


# ---------------------------------------------------------------------------------------------------------------
# Linear attention with a decay for each head, and the norms that join a block to the residual stream
# ---------------------------------------------------------------------------------------------------------------

# The descriptors as the C structs lie in memory; a call's own is packed, which takes a tenth of filling a ctypes object.
_LA_DESC, _LA_GRADS = struct.Struct("@8if12q"), struct.Struct("@12q")
_LA_STEP, _BN_DESC = struct.Struct("@8if9q"), struct.Struct("@q8i2fi3q")


def _on_stream(f):
    """Adds `stream`: the call and its buffers belong to that stream (torch's, or a raw handle), as under torch.cuda.stream."""
    @functools.wraps(f)
    def call(*args, stream=None, **kw):
        if stream is None:
            return f(*args, **kw)
        import torch
        if isinstance(stream, int):
            lead = next(a for a in (*args, *kw.values()) if isinstance(a, torch.Tensor))
            stream = torch.cuda.ExternalStream(stream, device=lead.device)
        with torch.cuda.stream(stream):
            return f(*args, **kw)
    return call


def _current(index):
    """The device's current stream, raw."""
    import torch
    return torch._C._cuda_getCurrentRawStream(index)


def _io_of(t, what):
    import torch
    if t.dtype == torch.float32:
        return 0
    if t.dtype == torch.bfloat16:
        return 1
    raise ValueError(f"{what} must be float32 or bfloat16, not {t.dtype}")


def _need_cuda(t, what):
    if t.device.type != "cuda":
        raise ValueError(f"{what} needs CUDA tensors (there is no CPU path)")


def _heads_like(like, B, H, L, D, dtype):
    """An empty [B][H][L][D] tensor whose memory is ordered like `like`'s: [B][L][H][D] where its positions are outermost."""
    if like.stride(2) > like.stride(1) and H > 1:
        return like.new_empty_strided((B, H, L, D), (L * H * D, D, H * D, 1), dtype=dtype)
    return like.new_empty((B, H, L, D), dtype=dtype)


def _unit(t):
    """The tensor with contiguous last axis (a copy where it is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _plain(t):
    """(contiguous tensor, its address), or None twice."""
    if t is None:
        return None, None
    t = t if t.is_contiguous() else t.contiguous()
    return t, t.data_ptr()


def check_linear_attention(q, k, v, log_decay, scale, initial_state, lengths, final_grad=None):
    """Raises ValueError where the arguments of linear_attention do not fit each other; else (B, H, L, D, Hkv, Dv, io)."""
    import torch
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k and v must be [B][H][L][D], [B][Hkv][L][D] and [B][Hkv][L][Dv]")
    (B, H, L, D), Hkv, Dv = q.shape, k.shape[1], v.shape[3]
    if k.shape != (B, Hkv, L, D) or v.shape != (B, Hkv, L, Dv):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if H < 1 or Hkv < 1 or H % Hkv:
        raise ValueError(f"{H} query heads cannot share {Hkv} key and value heads evenly")
    if D < 1 or Dv < 1:
        raise ValueError("head sizes must be positive")
    io = _io_of(q, "q")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have one type")
    if log_decay.shape != (H,) or log_decay.dtype != torch.float32:
        raise ValueError(f"log_decay must be a float32 [{H}] tensor")
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError("log_decay is a constant: it has no gradient (pass log_decay.detach())")
    if not math.isfinite(scale) or scale == 0:
        raise ValueError("scale must be finite and not 0")
    for t, what in ((initial_state, "initial_state"), (final_grad, "the final state's gradient")):
        if t is not None and (t.shape != (B, H, D, Dv) or t.dtype != torch.float32):
            raise ValueError(f"{what} must be a float32 {[B, H, D, Dv]} tensor")
    if lengths is not None and (lengths.shape != (B,) or lengths.dtype != torch.int32):
        raise ValueError(f"lengths must be an int32 [{B}] tensor")
    for t in (k, v, log_decay, initial_state, lengths, final_grad):
        if t is not None and t.device != q.device:
            raise ValueError("all tensors must be on one device")
    return B, H, L, D, Hkv, Dv, io


def _la_workspace(desc, backward, device):
    import torch
    need = ctypes.c_size_t()
    _check(lib().sffft_linear_attention_workspace_bytes(desc, backward, ctypes.byref(need)), "linear_attention_workspace_bytes")
    work = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
    return work, _ptr(work), need.value


@_on_stream
def linear_attention(q, k, v, log_decay, scale=1.0, initial_state=None, lengths=None):
    """(y, final_state) of S_n = lambda S_{n-1} + k_n v_n^T, y_n = scale S_n^T q_n, lambda = exp(log_decay) for each head.

    q [B][H][L][D], k [B][Hkv][L][D], v [B][Hkv][L][Dv], float32 or bfloat16; log_decay [H] float32, <= 0;
    initial_state and final_state [B][H][D][Dv] float32; lengths [B] int32: tokens of each row (default L).  y has
    q's type and order of axes, and is zero behind a row's last token.  Runs on `stream` (default: the current one)."""
    import torch
    B, H, L, D, Hkv, Dv, io = check_linear_attention(q, k, v, log_decay, scale, initial_state, lengths)
    _need_cuda(q, "linear_attention")
    q, k, v, dev = _unit(q), _unit(k), _unit(v), q.device
    y = _heads_like(q, B, H, L, Dv, q.dtype)
    s1 = q.new_empty((B, H, D, Dv), dtype=torch.float32)
    desc = _LA_DESC.pack(B, H, Hkv, L, D, Dv, io, dev.index, scale, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                         *y.stride()[:3])
    work, wp, wn = _la_workspace(desc, 0, dev)
    (ld, ldp), (s0, s0p), (ln, lnp) = _plain(log_decay), _plain(initial_state), _plain(lengths)
    _check(lib().sffft_linear_attention(desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), ldp, lnp, s0p, y.data_ptr(),
                                        s1.data_ptr(), wp, wn, _current(dev.index)), "linear_attention")
    return y, s1


@_on_stream
def linear_attention_backward(q, k, v, log_decay, dy, dfinal_state=None, scale=1.0, initial_state=None, lengths=None):
    """(dq, dk, dv, dinitial_state) of linear_attention; dinitial_state is None where there was no initial state."""
    import torch
    B, H, L, D, Hkv, Dv, io = check_linear_attention(q, k, v, log_decay, scale, initial_state, lengths, dfinal_state)
    _need_cuda(q, "linear_attention_backward")
    if dy.shape != (B, H, L, Dv) or dy.dtype != q.dtype or dy.device != q.device:
        raise ValueError(f"dy must be a {q.dtype} {[B, H, L, Dv]} tensor on q's device")
    q, k, v, dev = _unit(q), _unit(k), _unit(v), q.device
    if dy.stride(-1) != 1 or 0 in dy.stride():   # a sum's gradient comes expanded
        dy = dy.contiguous()
    dq, dk = _heads_like(q, B, H, L, D, q.dtype), _heads_like(k, B, Hkv, L, D, q.dtype)
    dv = _heads_like(v, B, Hkv, L, Dv, q.dtype)
    ds0 = None if initial_state is None else q.new_empty((B, H, D, Dv), dtype=torch.float32)
    desc = _LA_DESC.pack(B, H, Hkv, L, D, Dv, io, dev.index, scale, *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], 0, 0, 0)
    grads = _LA_GRADS.pack(*dy.stride()[:3], *dq.stride()[:3], *dk.stride()[:3], *dv.stride()[:3])
    work, wp, wn = _la_workspace(desc, 1, dev)
    (ld, ldp), (s0, s0p), (ln, lnp), (ds1, ds1p) = (_plain(t) for t in (log_decay, initial_state, lengths, dfinal_state))
    _check(lib().sffft_linear_attention_backward(
        desc, grads, q.data_ptr(), k.data_ptr(), v.data_ptr(), ldp, lnp, s0p, dy.data_ptr(), ds1p, dq.data_ptr(), dk.data_ptr(),
        dv.data_ptr(), _ptr(ds0), wp, wn, _current(dev.index)), "linear_attention_backward")
    return dq, dk, dv, ds0


def linear_attention_check(device: int = 0):
    """Waits for the device and raises if one of its linear attention kernels reported a device-side error, and clears it.
    Until then later calls raise the same, without waiting for a device."""
    _check(lib().sffft_linear_attention_check(device), "device status")


@_on_stream
def linear_attention_step(q, k, v, log_decay, state, slots=None, scale=1.0):
    """One token for each row: state[slot] <- lambda state[slot] + k v^T in place, y = scale state[slot]^T q.

    q [B][H][D], k [B][Hkv][D], v [B][Hkv][Dv]; state [pool][H][D][Dv] float32, of which only the slots' axis may have a
    stride of its own; slots [B] int32 (default: row b uses slot b).  A slot outside the pool marks a padded row, whose
    y is zero; so does a slot that an earlier row of the call has."""
    import torch
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k and v must be [B][H][D], [B][Hkv][D] and [B][Hkv][Dv]")
    (B, H, D), Hkv, Dv = q.shape, k.shape[1], v.shape[2]
    if k.shape != (B, Hkv, D) or v.shape != (B, Hkv, Dv):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if H < 1 or Hkv < 1 or H % Hkv:
        raise ValueError(f"{H} query heads cannot share {Hkv} key and value heads evenly")
    if D < 1 or Dv < 1:
        raise ValueError("head sizes must be positive")
    io = _io_of(q, "q")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have one type")
    if log_decay.shape != (H,) or log_decay.dtype != torch.float32:
        raise ValueError(f"log_decay must be a float32 [{H}] tensor")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if state.dim() != 4 or state.shape[1:] != (H, D, Dv) or state.dtype != torch.float32:
        raise ValueError(f"state must be a float32 [pool, {H}, {D}, {Dv}] tensor")
    pool, stride = state.shape[0], state.stride()
    if not state[0:1].is_contiguous() or (pool > 1 and stride[0] < H * D * Dv):
        raise ValueError("a slot's state must be contiguous and slots must not overlap")
    if slots is not None and (slots.shape != (B,) or slots.dtype != torch.int32):
        raise ValueError(f"slots must be an int32 [{B}] tensor")
    if slots is None and pool < B:
        raise ValueError(f"{B} rows need {B} slots")
    dev = q.device
    for t in (k, v, log_decay, state, slots):
        if t is not None and t.device != dev:
            raise ValueError("all tensors must be on one device")
    _need_cuda(q, "linear_attention_step")
    q, k, v = _unit(q), _unit(k), _unit(v)
    y = q.new_empty((B, H, Dv))
    d = _LA_STEP.pack(B, H, Hkv, D, Dv, pool, io, dev.index, scale, *q.stride()[:2], *k.stride()[:2], *v.stride()[:2], H * Dv, Dv,
                      stride[0])
    (ld, ldp), (sl, slp) = _plain(log_decay), _plain(slots)
    _check(lib().sffft_linear_attention_step(d, q.data_ptr(), k.data_ptr(), v.data_ptr(), ldp, state.data_ptr(), slp,
                                             y.data_ptr(), _current(dev.index)), "linear_attention_step")
    return y


def check_block_norm(x, y, gate, post_weight, weight, scale, eps, groups, act, dim):
    """Raises ValueError where the arguments of block_norm do not fit each other; else (channels, kind of gate, whether the
    layout is [B][C][L])."""
    import torch
    lead = y if y is not None else x
    if lead is None:
        raise ValueError("block_norm needs x or y")
    nd = lead.dim()
    if dim not in (-1, 1, nd - 1):
        raise ValueError("dim must be -1, or 1 for [B][C][L] tensors")
    first = dim == 1 and nd != 2
    if first and nd != 3:
        raise ValueError("dim 1 is for [B][C][L] tensors")
    if nd < 1 or lead.shape[dim] < 1:
        raise ValueError("there must be channels")
    C, dt, dev = lead.shape[dim], lead.dtype, lead.device
    if y is None:
        if gate is not None or post_weight is not None:
            raise ValueError("a gate and post_weight act on y")
        if weight is None:
            raise ValueError("without y there must be a weight to norm x with")
    if dt != torch.float32 and dt != torch.bfloat16:
        raise ValueError(f"the tensors must be float32 or bfloat16, not {dt}")
    if x is not None and y is not None:
        if x.shape != y.shape:
            raise ValueError(f"x {tuple(x.shape)} and y {tuple(y.shape)} must have one shape")
        if x.dtype != dt and x.dtype != torch.float32:
            raise ValueError("x must have y's type, or be float32 beside bfloat16")
        if x.device != dev:
            raise ValueError("all tensors must be on one device")
    kind = "none"
    if gate is not None:
        kind = "full" if gate.shape == y.shape else "channel"
        if kind == "channel" and gate.shape != (C,):
            raise ValueError(f"gate must be shaped like y or [{C}]")
        if gate.dtype != dt:
            raise ValueError("gate must have y's type")
        if gate.device != dev:
            raise ValueError("all tensors must be on one device")
    for w, what in ((post_weight, "post_weight"), (weight, "weight")):
        if w is not None:
            if w.shape != (C,):
                raise ValueError(f"{what} must be [{C}]")
            if w.dtype != torch.float32 and w.dtype != torch.bfloat16:
                raise ValueError(f"{what} must be float32 or bfloat16, not {w.dtype}")
            if w.device != dev:
                raise ValueError("all tensors must be on one device")
    if post_weight is not None and weight is not None and post_weight.dtype != weight.dtype:
        raise ValueError("the weights must have one type")
    if groups < 1 or C % groups:
        raise ValueError(f"{C} channels do not fall into {groups} groups")
    if act not in ACT:
        raise ValueError(f"act must be one of {sorted(ACT)}")
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if not math.isfinite(eps) or eps < 0:
        raise ValueError("eps must be finite and not negative")
    return C, kind, first


def _packed_like(t):
    """An empty contiguous tensor of t's shape and type."""
    import torch
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _as_rows(t, C):
    """(tensor, stride of a row) of a [..., C] tensor whose rows are evenly spaced (a copy where they are not)."""
    if t.is_contiguous():
        return t, C
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return t.contiguous(), C
    step, rows = None, 1
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if step is None:
            step = s
        elif s != step * rows:
            return t.contiguous(), C
        rows *= n
    return t, C if step is None else step


def _norm_desc(x, y, gate, post_weight, weight, scale, eps, groups, act, dim):
    """(descriptor, x, y, gate, weights, the tensor that the outputs are like, kind of gate, rows)"""
    import torch
    C, kind, first = check_block_norm(x, y, gate, post_weight, weight, scale, eps, groups, act, dim)
    lead = y if y is not None else x
    _need_cuda(lead, "block_norm")
    xs = ys = gs = 0
    if first:
        x, y, gate = (t if t is None or t.is_contiguous() else t.contiguous() for t in (x, y, gate))
    else:
        if x is not None:
            x, xs = _as_rows(x, C)
        if y is not None:
            y, ys = _as_rows(y, C)
        if kind == "full":
            gate, gs = _as_rows(gate, C)
        elif gate is not None and not gate.is_contiguous():
            gate = gate.contiguous()
    pw, w = (t if t is None or t.is_contiguous() else t.contiguous() for t in (post_weight, weight))
    some = pw if pw is not None else w
    bf = torch.bfloat16
    rows = lead.numel() // C
    d = _BN_DESC.pack(rows, C, lead.shape[2] if first else 0, groups, lead.dtype == bf, (lead if x is None else x).dtype == bf,
                      some is not None and some.dtype == bf, GATE[kind], ACT[act], scale, eps, lead.device.index, xs, ys, gs)
    return d, x, y, gate, pw, w, lead, kind, rows


@_on_stream
def block_norm(x=None, y=None, gate=None, post_weight=None, weight=None, scale=1.0, eps=1e-6, groups=1, act="none", dim=-1,
               stats=False):
    """(h, n) with a = y rstd_g(y) post_weight, h = x + scale act(gate) a, n = h rstd(h) weight, each part only where its
    tensor is given; rstd(z) = (mean z^2 + eps)^-1/2 over the channels (over each of `groups` runs of them for y,
    which says nothing without post_weight).

    The channels are the last axis, or axis 1 of [B][C][L] tensors (`dim=1`, the layout of the convolution).  gate: shaped
    like y, or [C]; act: "none", "silu" or "sigmoid".  y, gate and n have one type (float32 or bfloat16); x and h have it
    too, or are float32.  Without y, h is x; without weight, n is None.  `stats=True` also returns the rstd of y's groups
    and of h, for block_norm_backward.  Runs on `stream` (default: the current one)."""
    import torch
    given = x
    d, x, y, gate, pw, w, lead, _, rows = _norm_desc(x, y, gate, post_weight, weight, scale, eps, groups, act, dim)
    dev = lead.device
    h = given if y is None else _packed_like(lead if x is None else x)
    n = None if w is None else _packed_like(lead)
    r1 = lead.new_empty((rows, groups), dtype=torch.float32) if stats and pw is not None else None
    r2 = lead.new_empty((rows,), dtype=torch.float32) if stats and w is not None else None
    if rows:
        _check(lib().sffft_block_norm(d, _ptr(x), _ptr(y), _ptr(gate), _ptr(pw), _ptr(w), _ptr(h), _ptr(n), _ptr(r1), _ptr(r2),
                                      _current(dev.index)), "block_norm")
    return (h, n, r1, r2) if stats else (h, n)


@_on_stream
def block_norm_backward(dh, dn, x=None, y=None, gate=None, post_weight=None, weight=None, rstd_post=None, rstd=None,
                        scale=1.0, eps=1e-6, groups=1, act="none", dim=-1):
    """(dx, dy, dgate, dpost_weight, dweight) of block_norm from the gradients of h (None: zero) and n; None where the tensor
    was not given."""
    import torch
    d, x, y, gate, pw, w, lead, kind, rows = _norm_desc(x, y, gate, post_weight, weight, scale, eps, groups, act, dim)
    if (dn is None) != (w is None):
        raise ValueError("dn is needed where there is a weight, and only there")
    if dn is not None and (dn.shape != lead.shape or dn.dtype != lead.dtype):
        raise ValueError("dn must be like n")
    if dh is not None and (dh.shape != lead.shape or dh.dtype != (lead if x is None else x).dtype):
        raise ValueError("dh must be like h")
    if dh is None and w is None:
        raise ValueError("dh or dn is needed")
    for t, w_, n, what in ((rstd_post, pw, rows * groups, "rstd_post"), (rstd, w, rows, "rstd")):
        if w_ is not None and (t is None or t.numel() != n or t.dtype != torch.float32 or not t.is_contiguous()):
            raise ValueError(f"{what} must be the forward pass's")
    for t in (dh, dn, rstd_post, rstd):
        if t is not None and t.device != lead.device:
            raise ValueError("all tensors must be on one device")
    dh, dn = (t if t is None or t.is_contiguous() else t.contiguous() for t in (dh, dn))
    dev = lead.device
    dx, dy, dgate, dpw, dw = (None if t is None else _packed_like(t) for t in (x, y, gate, pw, w))
    if not rows:   # empty buffers have no address to pass
        for t in (dgate if kind == "channel" else None, dpw, dw):
            if t is not None:
                t.zero_()
        return dx, dy, dgate, dpw, dw
    need = ctypes.c_size_t()
    _check(lib().sffft_block_norm_workspace_bytes(d, ctypes.byref(need)), "block_norm_workspace_bytes")
    work = torch.empty(need.value, dtype=torch.uint8, device=dev) if need.value else None
    _check(lib().sffft_block_norm_backward(
        d, _ptr(x), _ptr(y), _ptr(gate), _ptr(pw), _ptr(w), _ptr(rstd_post), _ptr(rstd), _ptr(dh), _ptr(dn), _ptr(dx), _ptr(dy),
        _ptr(dgate), _ptr(dpw), _ptr(dw), _ptr(work), need.value, _current(dev.index)), "block_norm_backward")
    return dx, dy, dgate, dpw, dw
