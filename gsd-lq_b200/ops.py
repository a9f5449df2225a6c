"""Torch-tensor wrappers over the C ABI (device memory in, device memory out).

Every function launches on the current torch CUDA stream and raises
``GsdlqError`` when the library reports a failure.  No function here has a
CPU path.
"""
from __future__ import annotations

import ctypes
import math
import warnings

import numpy as np
import torch

from . import _lib as L
from .gsd2 import HexTensor


def ptr(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream_handle(stream: torch.cuda.Stream | None = None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _lib():
    return L.load()


def to_device_bytes(a: np.ndarray, device) -> torch.Tensor:
    """Upload the raw bytes of a NumPy array (any dtype) as a uint8 device tensor."""
    a = np.ascontiguousarray(a)
    t = torch.from_numpy(a.reshape(-1).view(np.uint8))
    return t.to(device, non_blocking=False)


class DeviceHex:
    """A packed linear resident in device memory (reference layout), with its C descriptor."""

    def __init__(self, t: HexTensor | None = None, device="cuda", arena: "Arena | None" = None, **tensors):
        if t is not None:
            self.rows, self.cols, self.k_dim, self.radius = t.rows, t.cols, t.k_dim, t.radius
            up = (lambda a: arena.put(a)) if arena is not None else (lambda a: to_device_bytes(a, device))
            self.codes = up(t.codes)
            self.scales = up(t.scales)
            self.row_ptr = up(t.row_ptr)
            self.kink_cols = up(t.kink_cols) if t.nnz else None
            self.kink_deltas = up(t.kink_deltas) if t.nnz else None
            self.U = up(t.U) if t.k_dim else None
            self.S = up(t.S) if t.k_dim else None
            self.Vt = up(t.Vt) if t.k_dim else None
            self.nnz = t.nnz
        else:  # already on the device (GPU packer)
            for k, v in tensors.items():
                setattr(self, k, v)
        self.n_pts = 217 if self.radius == 8 else 127

    def nbytes(self) -> int:
        n = 0
        for k in ("codes", "scales", "row_ptr", "kink_cols", "kink_deltas", "U", "S", "Vt"):
            v = getattr(self, k, None)
            if v is not None:
                n += v.numel() * v.element_size()
        return n

    def build_unit_kinks(self):
        """Regroup the CSR kinks per 16-row x 512-column work unit (gsdlq_unit_kinks); the fused
        linear then applies them in its streaming loop.  Keeps the CSR arrays (the drop-in path)."""
        gu = (self.cols // 64 + 7) // 8
        n_units = ((self.rows + 15) // 16) * gu
        dev = self.codes.device
        self.unit_kink_off = torch.zeros(n_units + 1, dtype=torch.int32, device=dev)
        self.unit_kinks = torch.zeros(max(1, 2 * self.nnz), dtype=torch.int32, device=dev)
        L.check(_lib().gsdlq_unit_kinks(ptr(self.row_ptr), ptr(self.kink_cols), ptr(self.kink_deltas), self.rows,
                                        self.cols, ptr(self.unit_kink_off), ptr(self.unit_kinks), stream_handle()),
                "gsdlq_unit_kinks")
        return self

    def desc(self) -> L.HexMat:
        uko = getattr(self, "unit_kink_off", None)
        uk = getattr(self, "unit_kinks", None)
        return L.HexMat(unit_kink_off=uko.data_ptr() if uko is not None else None,
                        unit_kinks=uk.data_ptr() if uk is not None else None,
                        codes=self.codes.data_ptr(), scales=self.scales.data_ptr(),
                        U=self.U.data_ptr() if self.U is not None else None,
                        S=self.S.data_ptr() if self.S is not None else None,
                        Vt=self.Vt.data_ptr() if self.Vt is not None else None,
                        row_ptr=self.row_ptr.data_ptr(),
                        kink_cols=self.kink_cols.data_ptr() if self.kink_cols is not None else None,
                        kink_deltas=self.kink_deltas.data_ptr() if self.kink_deltas is not None else None,
                        rows=self.rows, cols=self.cols, k_dim=self.k_dim, radius=self.radius)


class Arena:
    """One device allocation holding many 256-byte-aligned blobs (fewer, larger copies)."""

    ALIGN = 256

    def __init__(self, nbytes: int, device="cuda"):
        self.buf = torch.empty(nbytes + self.ALIGN, dtype=torch.uint8, device=device)
        self.off = (-self.buf.data_ptr()) % self.ALIGN
        self.cap = nbytes + self.ALIGN

    @classmethod
    def bytes_needed(cls, arrays) -> int:
        return sum((a.nbytes + cls.ALIGN - 1) // cls.ALIGN * cls.ALIGN for a in arrays)

    def put(self, a: np.ndarray) -> torch.Tensor:
        a = np.ascontiguousarray(a)
        n = a.nbytes
        if self.off + n > self.cap:
            raise MemoryError("arena overflow")
        dst = self.buf[self.off:self.off + n]
        if n:
            # read-only memory-mapped blobs go straight to the device: torch only reads the view
            with warnings.catch_warnings():
                warnings.filterwarnings("ignore", message="The given NumPy array is not writable")
                src = torch.from_numpy(a.reshape(-1).view(np.uint8))
            dst.copy_(src, non_blocking=False)
        self.off += (n + self.ALIGN - 1) // self.ALIGN * self.ALIGN
        return dst

    def alloc(self, n: int) -> torch.Tensor:
        if self.off + n > self.cap:
            raise MemoryError("arena overflow")
        dst = self.buf[self.off:self.off + n]
        self.off += (n + self.ALIGN - 1) // self.ALIGN * self.ALIGN
        return dst


# ---- drop-in functions (reference signatures) --------------------------------------------
def rmsnorm(x, w, out, eps):
    L.check(_lib().gsdlq_rmsnorm(ptr(x), ptr(w), ptr(out), x.numel(), eps, stream_handle()), "rmsnorm")


def vec_add(y, a, b):
    L.check(_lib().gsdlq_vec_add(ptr(y), ptr(a), ptr(b), y.numel(), stream_handle()), "vec_add")


def swiglu(gate, up, out):
    L.check(_lib().gsdlq_swiglu(ptr(gate), ptr(up), ptr(out), gate.numel(), stream_handle()), "swiglu")


def lowrank_proj(x, h: DeviceHex, tmp_k):
    L.check(_lib().gsdlq_lowrank_proj(ptr(x), ptr(h.Vt), ptr(h.S), ptr(tmp_k), h.k_dim, h.cols,
                                      stream_handle()), "lowrank_proj")


def hex2d_matvec(x, h: DeviceHex, xy_table, tmp_k, y):
    L.check(_lib().gsdlq_hex2d_matvec(ptr(x), ptr(h.codes), ptr(h.scales), ptr(xy_table), ptr(h.U), ptr(tmp_k),
                                      ptr(h.row_ptr), ptr(h.kink_cols), ptr(h.kink_deltas), ptr(y), h.rows, h.cols,
                                      h.k_dim, h.n_pts, stream_handle()), "hex2d_matvec")


MATMUL_MAX_BATCH = 128  # GSDLQ_MATMUL_MAX_BATCH


def matmul_work_bytes(batch: int, cols: int) -> int:
    n = ctypes.c_size_t()
    L.check(_lib().gsdlq_hex2d_matmul_work_size(batch, cols, ctypes.byref(n)), "hex2d_matmul_work_size")
    return int(n.value)


def matmul_work(batch: int, cols: int, device="cuda") -> torch.Tensor:
    """Scratch for hex2d_matmul of up to ``batch`` tokens and ``cols`` columns (1024-byte aligned)."""
    return torch.empty(matmul_work_bytes(batch, cols) + 1024, dtype=torch.uint8, device=device)


def _aligned(work: torch.Tensor) -> tuple[int, int]:
    p = work.data_ptr()
    a = (p + 1023) & ~1023
    return a, work.numel() * work.element_size() - (a - p)


def hex2d_matmul(x, h: DeviceHex, xy_table, y, work):
    """y[b] = the packed linear of x[b] for every row b of x ([batch][cols] -> [batch][rows]); work: a
    matmul_work buffer."""
    wp, wb = _aligned(work)
    L.check(_lib().gsdlq_hex2d_matmul(ptr(x), x.shape[0], ptr(h.codes), ptr(h.scales), ptr(xy_table), ptr(h.U),
                                      ptr(h.S), ptr(h.Vt), ptr(h.row_ptr), ptr(h.kink_cols), ptr(h.kink_deltas),
                                      ptr(y), wp, wb, h.rows, h.cols, h.k_dim, h.n_pts, stream_handle()),
            "hex2d_matmul")


def sample_top_p(logits: torch.Tensor, temperature: float, top_p: float, u: float) -> int:
    """gsdlq_sample_top_p over a device logits vector with the uniform draw u; returns the pick."""
    n = logits.numel()
    b = ctypes.c_size_t()
    L.check(_lib().gsdlq_sample_work_size(n, ctypes.byref(b)), "sample_work_size")
    work = torch.empty(int(b.value), dtype=torch.uint8, device=logits.device)
    ud = torch.tensor([u], dtype=torch.float64, device=logits.device)
    out = torch.full((1,), -2, dtype=torch.int32, device=logits.device)
    L.check(_lib().gsdlq_sample_top_p(ptr(logits), n, float(temperature), float(top_p), ptr(ud), None, ptr(work),
                                      work.numel(), None, ptr(out), stream_handle()), "sample_top_p")
    return int(out.item())


def attention_rows_work(n: int, n_heads: int, head_dim: int, device="cuda") -> torch.Tensor:
    """Scratch for gsdlq_attention_rows of up to ``n`` tokens (float32; torch's allocations are 16-byte
    aligned)."""
    b = ctypes.c_size_t()
    L.check(_lib().gsdlq_attention_rows_work_size(n, n_heads, head_dim, ctypes.byref(b)), "attention_rows_work_size")
    return torch.empty(int(b.value), dtype=torch.uint8, device=device)


def rope_and_store_kv(q, k, v, k_cache, v_cache, layer, pos, n_heads, n_kv, hd, max_seq, theta, interleaved=1):
    L.check(_lib().gsdlq_rope_and_store_kv(ptr(q), ptr(k), ptr(v), ptr(k_cache), ptr(v_cache), layer, pos, n_heads,
                                           n_kv, hd, max_seq, theta, interleaved, stream_handle()),
            "rope_and_store_kv")


def gqa_attention(q, k_cache, v_cache, out, layer, pos, n_heads, n_kv, hd, max_seq, sm_scale):
    L.check(_lib().gsdlq_gqa_attention(ptr(q), ptr(k_cache), ptr(v_cache), ptr(out), layer, pos, n_heads, n_kv, hd,
                                       max_seq, sm_scale, stream_handle()), "gqa_attention")


# ---- engine functions ---------------------------------------------------------------------
def codebook(radius: int) -> np.ndarray:
    buf = np.zeros(2 * 256, np.float32)
    n = _lib().gsdlq_codebook(radius, buf.ctypes.data_as(ctypes.c_void_p), 256)
    if n < 0:
        L.check(n, "codebook")
    return buf[:2 * n].reshape(n, 2).copy()


def dequant(h: DeviceHex, xy_table, out):
    L.check(_lib().gsdlq_dequant(ptr(h.codes), ptr(h.scales), ptr(xy_table), ptr(out), h.rows, h.cols, h.n_pts,
                                 stream_handle()), "dequant")


def argmax(x, out_idx):
    L.check(_lib().gsdlq_argmax(ptr(x), x.numel(), ptr(out_idx), stream_handle()), "argmax")


def pack_lattice(w: torch.Tensor, radius: int, codes, scales, residual=None):
    r, c = w.shape
    L.check(_lib().gsdlq_pack_lattice(ptr(w), r, c, radius, ptr(codes), ptr(scales), ptr(residual),
                                      stream_handle()), "pack_lattice")


def rope_table(max_seq: int, head_dim: int, theta: float) -> np.ndarray:
    t = np.zeros((max_seq, head_dim // 2, 2), np.float32)
    L.check(_lib().gsdlq_rope_table(t.ctypes.data_as(ctypes.c_void_p), max_seq, head_dim, theta), "rope_table")
    return t


def linear_ws_size(job: L.LinearJob) -> int:
    n = ctypes.c_size_t(0)
    L.check(_lib().gsdlq_linear_ws_size(ctypes.byref(job), ctypes.byref(n)), "gsdlq_linear_ws_size")
    return n.value


def linear_workspace(job: L.LinearJob, device="cuda") -> torch.Tensor:
    """A zeroed, 16-byte aligned device workspace large enough for ``job``."""
    return torch.zeros((linear_ws_size(job) + 15) // 16 * 4, dtype=torch.int32, device=device)


def linear(job: L.LinearJob, ws: torch.Tensor):
    L.check(_lib().gsdlq_linear(ctypes.byref(job), ptr(ws), ws.numel() * ws.element_size(), stream_handle()),
            "gsdlq_linear")


def attention_ws_size(n_heads, n_kv, hd, max_seq) -> tuple[int, int]:
    pb, wb = ctypes.c_size_t(0), ctypes.c_size_t(0)
    L.check(_lib().gsdlq_attention_ws_size(n_heads, n_kv, hd, max_seq, ctypes.byref(pb), ctypes.byref(wb)),
            "attention_ws_size")
    return pb.value, wb.value


def attention(job: L.AttnJob):
    L.check(_lib().gsdlq_attention(ctypes.byref(job), stream_handle()), "gsdlq_attention")


# ---- paged cache and log probabilities ----------------------------------------------------
# The calls below take a job (the C descriptor with its tensors checked once and kept alive), as linear() and
# attention() do: a decode loop builds its jobs at the start and launches them every step.
def _check(t, name: str, dtype, shape, device, row_stride: bool = False):
    """A device tensor of the given dtype and shape (None: any size there) on ``device``; contiguous, but for
    the stride between its rows where ``row_stride``."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    if t.device != device or t.device.type != "cuda":
        raise ValueError(f"{name} must be on the CUDA device of the call ({device}), not on {t.device}")
    if t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)):
        raise ValueError(f"{name} must have shape {tuple(shape)}, not {tuple(t.shape)}")
    inner = t[0] if row_stride and t.shape[0] else t
    if not inner.is_contiguous() or (row_stride and t.shape[0] > 1 and t.stride(0) < inner.numel()):
        raise ValueError(f"{name} must be contiguous" + (" within its rows" if row_stride else ""))
    return t


def _row_stride(t, most: int = 2**31 - 1) -> int:
    """Elements between t's rows, for a descriptor that holds up to ``most`` (an int's)."""
    n = t.stride(0) if t.shape[0] > 1 else 0
    if n > most:
        raise ValueError(f"rows more than {most} elements apart")
    return n


def _ints(t, name: str, device, n: int | None = None) -> int:
    """_check of a vector of int32 (of n entries), for calls made every step; returns its length."""
    if not (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.dim() == 1 and t.device == device
            and t.is_contiguous() and (n is None or t.numel() == n)):
        _check(t, name, torch.int32, (n,), device)
    return t.numel()


def _rows(kv, pos, row_seq, device):
    rows = _ints(pos, "pos", device)
    if row_seq is not None:
        _ints(row_seq, "row_seq", device, rows)
    if rows < 1 or (row_seq is None and rows > kv.n_seqs):
        raise ValueError("one row per sequence without row_seq, and at least one")
    return rows


def _stream_on(device) -> int:
    """The current stream of the tensors' device, which must be the current one (launches go there)."""
    i = torch.cuda.current_device()
    if device.index != i:
        raise ValueError(f"the tensors are on {device}, but cuda:{i} is the current device")
    return torch._C._cuda_getCurrentRawStream(i)


def paged_append_job(kv, layer: int, q, k, v, q_out, pos, rope_cs, row_seq=None, interleaved: bool = True):
    """Job of rope_kv_paged: q [rows][heads][head_dim], k and v [rows][kv heads][head_dim] (fp32, rows may be
    strided, k and v alike), q_out like q (or q itself), rope_cs [positions][head_dim / 2][2]."""
    dev, hd = kv.k.device, kv.head_dim
    rows = _rows(kv, pos, row_seq, dev)
    _check(q, "q", torch.float32, (rows, None, hd), dev, row_stride=True)
    _check(q_out, "q_out", torch.float32, tuple(q.shape), dev, row_stride=True)
    for t, name in ((k, "k"), (v, "v")):
        _check(t, name, torch.float32, (rows, kv.n_kv_heads, hd), dev, row_stride=True)
    if _row_stride(k) != _row_stride(v):
        raise ValueError("k and v must have the same row stride")
    _check(rope_cs, "rope_cs", torch.float32, (None, hd // 2, 2), dev)
    if rope_cs.data_ptr() % 8:
        raise ValueError("rope_cs must start at a multiple of 8 bytes")
    if not 0 <= layer < kv.n_layers:
        raise ValueError(f"layer outside [0, {kv.n_layers})")
    j = L.PagedAppendJob(kv=kv.desc(), layer=layer, q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(),
                         q_out=q_out.data_ptr(), q_stride=_row_stride(q), kv_stride=_row_stride(k),
                         q_out_stride=_row_stride(q_out), rope_cs=rope_cs.data_ptr(), max_pos=rope_cs.shape[0],
                         interleaved=int(interleaved), row_seq=None if row_seq is None else row_seq.data_ptr(),
                         pos=pos.data_ptr(), rows=rows, n_heads=q.shape[1])
    j.keep, j.device = (kv, q, k, v, q_out, pos, rope_cs, row_seq), dev
    return j


def rope_kv_paged(job):
    """RoPE of the job's rows and their k and v into their pages (gsdlq_rope_kv_paged)."""
    status = _lib().gsdlq_rope_kv_paged(job, _stream_on(job.device))
    if status:
        L.check(status, "gsdlq_rope_kv_paged")


def attention_paged_work(kv, rows: int, n_heads: int) -> torch.Tensor:
    """A zeroed work area for attention_paged, shared by any jobs of up to ``rows`` rows that follow one another (one
    per launch that may overlap)."""
    n = ctypes.c_size_t()
    L.check(_lib().gsdlq_attention_paged_work_size(rows, n_heads, kv.n_kv_heads, kv.head_dim, ctypes.byref(n)),
            "attention_paged_work_size")
    return torch.zeros(int(n.value), dtype=torch.uint8, device=kv.k.device)


def paged_attn_job(kv, layer: int, q, out, pos, sm_scale: float, work, row_seq=None):
    """Job of attention_paged: q [rows][heads][head_dim] fp32 (rows may be strided), out the same shape, packed.

    Whether neighbouring rows of a sequence share their reads of K and V goes by the rows per sequence of the table.
    For a chunk of one sequence b out of many, make the job over a cache of that sequence alone, with a row_seq of
    zeros: PagedKV.wrap(kv.k, kv.v, kv.table[b:b + 1], kv.refs)."""
    dev, hd = kv.k.device, kv.head_dim
    rows = _rows(kv, pos, row_seq, dev)
    _check(q, "q", torch.float32, (rows, None, hd), dev, row_stride=True)
    _check(out, "out", torch.float32, tuple(q.shape), dev)
    _check(work, "work", torch.uint8, (None,), dev)
    if not 0 <= layer < kv.n_layers:
        raise ValueError(f"layer outside [0, {kv.n_layers})")
    if q.shape[1] < 1 or q.shape[1] % kv.n_kv_heads:
        raise ValueError("the query heads must be a multiple of the kv heads")
    if not math.isfinite(sm_scale):
        raise ValueError("sm_scale must be finite")
    if q.data_ptr() % 16 or _row_stride(q) % 4:
        raise ValueError("q and its rows must start at multiples of 16 bytes")
    j = L.PagedAttnJob(kv=kv.desc(), layer=layer, q=q.data_ptr(), q_stride=_row_stride(q), out=out.data_ptr(),
                       row_seq=None if row_seq is None else row_seq.data_ptr(), pos=pos.data_ptr(), rows=rows,
                       n_heads=q.shape[1], sm_scale=sm_scale, work=work.data_ptr(), work_bytes=work.numel())
    j.keep, j.device = (kv, q, out, pos, work, row_seq), dev
    return j


def attention_paged(job):
    """Attention of the job's rows over their sequences' pages (gsdlq_attention_paged)."""
    status = _lib().gsdlq_attention_paged(job, _stream_on(job.device))
    if status:
        L.check(status, "gsdlq_attention_paged")


def logprobs_job(logits, ids=None, logprob=None, entropy=None, top_ids=None, top_logprobs=None,
                 temperature: float = 1.0):
    """Job of logprobs_rows: logits [rows][n] fp32 (rows may be strided); ids int32 [rows] with logprob [rows];
    entropy [rows]; top_ids int32 and top_logprobs [rows][top].  What is None is not computed."""
    if not isinstance(logits, torch.Tensor):
        raise TypeError("logits must be a tensor")
    dev = logits.device
    _check(logits, "logits", torch.float32, (None, None), dev, row_stride=True)
    rows, n = logits.shape
    if rows < 1 or n < 1:
        raise ValueError("logits must have at least one row and one column")
    if (ids is None) != (logprob is None) or (top_ids is None) != (top_logprobs is None):
        raise ValueError("ids and logprob, and top_ids and top_logprobs, go together")
    if ids is None and entropy is None and top_ids is None:
        raise ValueError("nothing to compute")
    for t, name, dt in ((ids, "ids", torch.int32), (logprob, "logprob", torch.float32),
                        (entropy, "entropy", torch.float32)):
        if t is not None:
            _check(t, name, dt, (rows,), dev)
    top = 0
    if top_ids is not None:
        top = _check(top_ids, "top_ids", torch.int32, (rows, None), dev).shape[1]
        _check(top_logprobs, "top_logprobs", torch.float32, (rows, top), dev)
        if top > min(n, L.MAX_TOP):
            raise ValueError(f"at most {min(n, L.MAX_TOP)} alternatives")
    if not (temperature > 0.0 and math.isfinite(temperature)):
        raise ValueError("temperature must be positive and finite")
    opt = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    j = L.LogprobsJob(logits=logits.data_ptr(), row_stride=_row_stride(logits, 2**63 - 1), rows=rows, n=n,
                      temperature=temperature, ids=opt(ids), logprob=opt(logprob), entropy=opt(entropy), top=top,
                      top_ids=opt(top_ids), top_logprobs=opt(top_logprobs))
    j.keep, j.device = (logits, ids, logprob, entropy, top_ids, top_logprobs), dev
    return j


def logprobs_rows(job):
    """Log probabilities, entropy and top alternatives of the job's rows (gsdlq_logprobs_rows)."""
    status = _lib().gsdlq_logprobs_rows(job, _stream_on(job.device))
    if status:
        L.check(status, "gsdlq_logprobs_rows")
