"""torch-facing wrappers of the libtq_b200 C ABI.

Tensors are owned by PyTorch; the kernels borrow raw device pointers and run
on the current CUDA stream.  Every wrapper raises (never falls back to a CPU
or PyTorch implementation) when the library or the device is unavailable.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import struct
import threading
from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd import forward_ad

from .. import _lib

_DT = {torch.float32: _lib.TQ_F32, torch.float16: _lib.TQ_F16, torch.bfloat16: _lib.TQ_BF16}


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _require_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise RuntimeError("TurboQuant kernels need CUDA tensors (there is no CPU path)")


def tensor4(x: torch.Tensor) -> _lib.Tensor4:
    if x.dim() != 4:
        raise ValueError(f"expected a 4-d tensor, got shape {tuple(x.shape)}")
    if x.dtype not in _DT:
        raise ValueError(f"unsupported dtype {x.dtype}")
    t = _lib.Tensor4()
    t.data = x.data_ptr()
    t.dtype = _DT[x.dtype]
    t.shape[:] = x.shape
    t.stride[:] = x.stride()
    return t


@dataclass
class LayerTables:
    """Per-layer constant device tables (codebooks, rotation, QJL matrix)."""
    head_dim: int
    key_bits: int
    value_bits: int
    qjl: bool
    k_centroids: torch.Tensor
    k_boundaries: torch.Tensor
    v_centroids: torch.Tensor
    v_boundaries: torch.Tensor
    rot: torch.Tensor
    qjl_mat: Optional[torch.Tensor] = None
    rot_t: Optional[torch.Tensor] = None
    qjl_t: Optional[torch.Tensor] = None
    rot_bf16x3: Optional[torch.Tensor] = None
    rot_f16: Optional[torch.Tensor] = None
    qjl_bf16: Optional[torch.Tensor] = None

    def __post_init__(self):
        self.rot = self.rot.contiguous().float()
        if self.rot.data_ptr() % 16:                     # a slice of something larger
            self.rot = self.rot.clone()
        self.rot_t = self.rot.t().contiguous()
        self.rot_f16 = self.rot.half().contiguous()      # prefill attention
        if self.head_dim == 128:
            # R = hi + mid + lo in bf16 (24 significant bits): the tensor-core
            # append computes x R^T as three exact bf16 products summed in fp32;
            # rows permuted into the packed K / V orders (tq_tables.rot_bf16x3)
            hi = self.rot.bfloat16()
            r1 = self.rot - hi.float()
            mid = r1.bfloat16()
            lo = (r1 - mid.float()).bfloat16()
            terms = torch.stack([hi, mid, lo])
            ko, vo = row_orders(self.head_dim)
            dev = self.rot.device
            self.rot_bf16x3 = torch.stack([terms[:, torch.as_tensor(ko, device=dev)],
                                           terms[:, torch.as_tensor(vo, device=dev)]]).contiguous()
        if self.qjl_mat is not None:
            self.qjl_mat = self.qjl_mat.contiguous().float()
            self.qjl_t = self.qjl_mat.t().contiguous()
            # the tensor-core append sketches with S in bf16: only when S is
            # exactly bf16 (the library's own S is), rows and columns in K
            # quad order (tq_tables.qjl_bf16)
            sb = self.qjl_mat.bfloat16()
            if self.head_dim == 128 and torch.equal(sb.float(), self.qjl_mat):
                ko = torch.as_tensor(row_orders(self.head_dim)[0], device=self.qjl_mat.device)
                self.qjl_bf16 = sb[ko][:, ko].contiguous()

    def __setattr__(self, name, value):
        # a changed table invalidates the cached C descriptors
        self.__dict__.pop("_geom", None)
        self.__dict__.pop("_ctab", None)
        super().__setattr__(name, value)

    def geom(self) -> _lib.Geom:
        g = self.__dict__.get("_geom")
        if g is None:
            g = _lib.Geom(self.head_dim, self.key_bits, self.value_bits, 1 if self.qjl else 0)
            self.__dict__["_geom"] = g
        return g

    def ctables(self) -> _lib.Tables:
        """The C table descriptor (built once: the tables never move)."""
        t = self.__dict__.get("_ctab")
        if t is None:
            t = self._build_ctables()
            self.__dict__["_ctab"] = t
        return t

    def _build_ctables(self) -> _lib.Tables:
        t = _lib.Tables()
        t.k_centroids = self.k_centroids.data_ptr()
        t.k_boundaries = self.k_boundaries.data_ptr()
        t.v_centroids = self.v_centroids.data_ptr()
        t.v_boundaries = self.v_boundaries.data_ptr()
        t.rot = self.rot.data_ptr()
        t.qjl = self.qjl_mat.data_ptr() if self.qjl_mat is not None else None
        t.rot_t = self.rot_t.data_ptr()
        t.qjl_t = self.qjl_t.data_ptr() if self.qjl_t is not None else None
        t.rot_bf16x3 = self.rot_bf16x3.data_ptr() if self.rot_bf16x3 is not None else None
        t.rot_f16 = self.rot_f16.data_ptr() if self.rot_f16 is not None else None
        t.qjl_bf16 = self.qjl_bf16.data_ptr() if self.qjl_bf16 is not None else None
        return t


def row_orders(head_dim: int):
    """Coordinate stored at each position of a packed K row (quad order: quad t
    lists 16j+2t, 16j+2t+1, 16j+2t+8, 16j+2t+9 for every 16-coordinate chunk j)
    and of a packed V row (octet order: octet g lists g, g+8, g+16, ...)."""
    k = [16 * j + 2 * t + e for t in range(4) for j in range(head_dim // 16)
         for e in (0, 1, 8, 9)]
    v = [g + 8 * c for g in range(8) for c in range(head_dim // 8)]
    return k, v


def page_bytes(head_dim: int, key_bits: int, value_bits: int, qjl: bool) -> int:
    """Bytes of one 64-token page (same formula as tq_page_bytes)."""
    krow, vrow = head_dim * key_bits // 8, head_dim * value_bits // 8
    qrow = head_dim // 8 if qjl else 0
    return _lib.PAGE_TOKENS * (krow + vrow + qrow + 4 + (2 if qjl else 0))


@dataclass
class PagedPages:
    """Paged storage (vLLM-style): a pool of pages and one block table row per
    stream; logical page p of stream s is pool[block_table[s, p]].  Accepted
    wherever a contiguous (streams, pages, page_bytes) tensor is.  Entries
    outside the pool are never dereferenced: the kernels read pool page 0 /
    drop the write and set _lib.DEV_BAD_BLOCK in the device status word."""
    pool: torch.Tensor          # uint8 (num_blocks, page_bytes)
    block_table: torch.Tensor   # int32 (streams, max_pages)

    def __post_init__(self):
        if self.pool.dtype != torch.uint8 or self.pool.dim() != 2:
            raise ValueError("pool must be uint8 (num_blocks, page_bytes)")
        if self.block_table.dtype != torch.int32 or self.block_table.dim() != 2 or \
                self.block_table.stride(1) != 1:
            raise ValueError("block_table must be int32 (streams, max_pages), rows contiguous")
        if self.block_table.device != self.pool.device:
            raise ValueError("pool and block_table must be on the same device")

    @property
    def is_cuda(self) -> bool:
        return self.pool.is_cuda

    @property
    def device(self) -> torch.device:
        return self.pool.device

    @property
    def shape(self):
        """(streams, pages per stream, page_bytes), as a contiguous page tensor."""
        return (self.block_table.shape[0], self.block_table.shape[1], self.pool.shape[1])


def _cache_desc(pages) -> _lib.Cache:
    if isinstance(pages, PagedPages):
        bt = pages.block_table
        return _lib.Cache(pages.pool.data_ptr(), bt.shape[0], bt.shape[1], bt.data_ptr(),
                          bt.stride(0), pages.pool.shape[0])
    return _lib.Cache(pages.data_ptr(), pages.shape[0], pages.shape[1])


# ---------------------------------------------------------------------------
def quantize_rotated(y: torch.Tensor, boundaries: torch.Tensor) -> torch.Tensor:
    """Bit-exact torch.bucketize(y, boundaries) -> int16, on the GPU."""
    _require_cuda(y, boundaries)
    y = y.contiguous().float()
    b = boundaries.contiguous().float()
    codes = torch.empty(y.shape, dtype=torch.int16, device=y.device)
    lib = _lib.load()
    _lib.check("tq_quantize_rotated",
               lib.tq_quantize_rotated(y.data_ptr(), y.numel(), b.data_ptr(), b.numel(),
                                       codes.data_ptr(), _stream(y.device)))
    return codes


def append(tables: LayerTables, pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
           pos: int) -> None:
    """Quantise and store tokens [pos, pos+T) of (B, H, T, D) k/v into pages."""
    _require_cuda(pages, k, v)
    lib = _lib.load()
    g, t, c = tables.geom(), tables.ctables(), _cache_desc(pages)
    kt, vt = tensor4(k), tensor4(v)
    _lib.check("tq_append", lib.tq_append(ctypes.byref(g), ctypes.byref(t), ctypes.byref(c),
                                          ctypes.byref(kt), ctypes.byref(vt), int(pos),
                                          _stream(k.device)))


def append_uses_tensor_cores(tables: LayerTables, k: torch.Tensor, v: torch.Tensor) -> bool:
    """True when append() with these inputs runs the tcgen05 kernel."""
    lib = _lib.load()
    g, t = tables.geom(), tables.ctables()
    kt, vt = tensor4(k), tensor4(v)
    return bool(lib.tq_append_tensor_core(ctypes.byref(g), ctypes.byref(t), ctypes.byref(kt),
                                          ctypes.byref(vt)))


def device_status(device: Optional[torch.device] = None) -> int:
    """Read and clear the library's status word on ``device`` (by default the
    current one), an OR of _lib.DEV_* (0: no kernel had anything to report)."""
    lib = _lib.load()
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    st = ctypes.c_uint32(0)
    with _on(device):                                    # each device has a word of its own
        rc = lib.tq_device_status(ctypes.byref(st), _stream(device))
    if rc not in (_lib.TQ_OK, _lib.TQ_ERR_DEVICE):
        _lib.check("tq_device_status", rc)
    return int(st.value)


def dequantize(tables: LayerTables, pages: torch.Tensor, t0: int, t1: int,
               k_out: Optional[torch.Tensor], v_out: Optional[torch.Tensor]) -> None:
    """Write dequantised tokens [t0, t1) into (B, H, t1-t0, D) views."""
    _require_cuda(pages, k_out, v_out)
    lib = _lib.load()
    g, t, c = tables.geom(), tables.ctables(), _cache_desc(pages)
    ko = tensor4(k_out) if k_out is not None else None
    vo = tensor4(v_out) if v_out is not None else None
    _lib.check("tq_dequantize", lib.tq_dequantize(
        ctypes.byref(g), ctypes.byref(t), ctypes.byref(c), int(t0), int(t1),
        ctypes.byref(ko) if ko is not None else None,
        ctypes.byref(vo) if vo is not None else None, _stream(pages.device)))


def _capturing(device: torch.device) -> bool:
    return device.type == "cuda" and torch.cuda.is_current_stream_capturing()


class DecodeWorkspace:
    """Grow-only device scratch of the attention calls (first 4 bytes: status
    word), one call at a time: calls of one stream may share it, and so may
    graphs that are replayed on one stream.  A buffer that a captured call
    has been given is kept as long as the workspace, since every replay writes
    to it; keep the workspace as long as the graph."""

    def __init__(self):
        self.buf: Optional[torch.Tensor] = None
        self._captured = False      # a graph holds the address of buf
        self._unset = False         # allocated while capturing: zeroed by the graph's replay only
        self._kept = []             # earlier buffers whose address a graph holds

    def get(self, nbytes: int, device: torch.device) -> torch.Tensor:
        capturing = _capturing(device)
        if self.buf is None or self.buf.numel() < nbytes or self.buf.device != device:
            if self._captured:
                self._kept.append(self.buf)
            self.buf = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=device)
            self._captured, self._unset = False, capturing
        elif self._unset and not capturing:
            self.buf.zero_()
            self._unset = False
        self._captured = self._captured or capturing
        return self.buf

    def status(self) -> int:
        """Read and clear the device status word (synchronises the stream)."""
        if self.buf is None:
            return 0
        lib = _lib.load()
        st = ctypes.c_uint32(0)
        lib.tq_workspace_status(self.buf.data_ptr(), ctypes.byref(st), _stream(self.buf.device))
        return int(st.value)


def _seq_lens_ptr(seq_lens: Optional[torch.Tensor], q: torch.Tensor) -> Optional[int]:
    if seq_lens is None:
        return None
    if seq_lens.dtype != torch.int32 or seq_lens.dim() != 1 or \
            seq_lens.shape[0] != q.shape[0] or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous int32 (B,) tensor")
    if seq_lens.device != q.device:
        raise ValueError("seq_lens must be on the query's device")
    return seq_lens.data_ptr()


def _row_ptr(x: Optional[torch.Tensor], q: torch.Tensor, name: str) -> Optional[int]:
    """Device pointer of an int32 (B,) per-row tensor (seq_lens, kv_start)."""
    if x is None:
        return None
    if x.dtype != torch.int32 or x.dim() != 1 or x.shape[0] != q.shape[0] or \
            not x.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 (B,) tensor")
    if x.device != q.device:
        raise ValueError(f"{name} must be on the query's device")
    return x.data_ptr()


def _decode_args(q, out, n_tokens, window_k, window_v, scale, num_ctas, phases, keep,
                 seq_lens=None, kv_start=None):
    qt, ot = tensor4(q), tensor4(out)
    wk = tensor4(window_k) if window_k is not None and window_k.shape[2] > 0 else None
    wv = tensor4(window_v) if wk is not None else None
    keep += [qt, ot, wk, wv]
    a = _lib.DecodeArgs()
    a.q = ctypes.pointer(qt)
    a.out = ctypes.pointer(ot)
    a.window_k = ctypes.pointer(wk) if wk is not None else None
    a.window_v = ctypes.pointer(wv) if wv is not None else None
    a.n_tokens = int(n_tokens)
    a.num_q_heads = q.shape[1]
    a.scale = float(scale if scale is not None else 1.0 / math.sqrt(q.shape[-1]))
    a.num_ctas = int(num_ctas)
    a.phases = int(phases)
    a.seq_lens = _seq_lens_ptr(seq_lens, q)
    a.kv_start = _row_ptr(kv_start, q, "kv_start")
    return a


def decode_step(tables: LayerTables, pages: torch.Tensor, k_new: torch.Tensor,
                v_new: torch.Tensor, pos: int, q: torch.Tensor,
                window_k: Optional[torch.Tensor] = None,
                window_v: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                out: Optional[torch.Tensor] = None,
                workspace: Optional[DecodeWorkspace] = None,
                num_ctas: int = 0, gather: Optional[_lib.Gather] = None,
                seq_lens: Optional[torch.Tensor] = None,
                kv_start: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Store the new (B, Hkv, 1, D) token at ``pos`` and attend q over tokens
    [0, pos + 1) plus the window, in one call (tq_decode_step).  ``gather``
    (a filled _lib.Gather whose peer_out[rank] is ``out``) also delivers the
    output block to every rank's gathered buffer (fused all-gather).

    ``seq_lens`` (int32 (B,) on the device, each <= pos + 1) makes the batch
    ragged: row b stores its token at seq_lens[b] - 1 and attends tokens
    [0, seq_lens[b]); ``pos`` is then the bound (the longest row's position).
    ``kv_start`` (int32 (B,) on the device): row b's keys before that position
    take no weight (left padding)."""
    _require_cuda(pages, q, k_new, v_new)
    lib = _lib.load()
    if out is None:
        out = torch.empty_like(q)
    g, t, c = tables.geom(), tables.ctables(), _cache_desc(pages)
    keep = []
    a = _decode_args(q, out, pos + 1, window_k, window_v, scale, num_ctas, 0, keep, seq_lens,
                     kv_start)
    if gather is not None:
        a.gather = ctypes.pointer(gather)
    kt, vt = tensor4(k_new), tensor4(v_new)
    nbytes = lib.tq_decode_workspace_bytes(ctypes.byref(g), ctypes.byref(c), ctypes.byref(a))
    if nbytes == 0:
        raise _lib.TqError("tq_decode_workspace_bytes", _lib.TQ_ERR_INVALID, _lib.last_error())
    ws = (workspace or DecodeWorkspace()).get(nbytes, q.device)
    _lib.check("tq_decode_step", lib.tq_decode_step(
        ctypes.byref(g), ctypes.byref(t), ctypes.byref(c), ctypes.byref(kt), ctypes.byref(vt),
        int(pos), ctypes.byref(a), ws.data_ptr(), ws.numel(), _stream(q.device)))
    return out


def prefill_uses_tensor_cores(tables: LayerTables) -> bool:
    """Whether prefill_attention (engine 0) runs the tcgen05 kernel for this
    layer's geometry."""
    return bool(_lib.load().tq_prefill_tensor_core(ctypes.byref(tables.geom())))


def prefill_attention(tables: LayerTables, pages: torch.Tensor, q: torch.Tensor,
                      n_tokens: int, scale: Optional[float] = None, causal: bool = True,
                      out: Optional[torch.Tensor] = None, engine: int = 0,
                      kv_start: Optional[torch.Tensor] = None,
                      window_k: Optional[torch.Tensor] = None,
                      window_v: Optional[torch.Tensor] = None,
                      workspace: Optional[DecodeWorkspace] = None) -> torch.Tensor:
    """Attention of queries q (B, Hq, Tq, D) at positions n_tokens - Tq ..
    n_tokens - 1 over the packed tokens [0, n_tokens) of every stream (causal:
    a query sees keys at or before its position).  ``engine`` 0 picks the
    fastest kernel (tcgen05 where prefill_uses_tensor_cores), 1 the mma.sync
    kernel, 2 / 3 the tcgen05 kernel with 128 / 256 query rows per CTA.
    ``kv_start`` (int32 (B,) on the device): row b's keys before that position
    take no weight (left padding; a query with no key left returns zeros).
    ``window_k`` / ``window_v`` ((B, Hkv, W, D)): the residual window, dense
    keys at positions n_tokens - W .. n_tokens - 1 after the packed ones."""
    _require_cuda(pages, q)
    lib = _lib.load()
    if out is None:
        out = torch.empty_like(q)
    g, t, c = tables.geom(), tables.ctables(), _cache_desc(pages)
    qt, ot = tensor4(q), tensor4(out)
    a = _lib.PrefillArgs(ctypes.pointer(qt), ctypes.pointer(ot), int(n_tokens),
                         float(scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])),
                         1 if causal else 0, int(engine), _row_ptr(kv_start, q, "kv_start"))
    if window_k is not None and window_k.shape[2] > 0:
        wk, wv = tensor4(window_k), tensor4(window_v)
        a.window_k, a.window_v = ctypes.pointer(wk), ctypes.pointer(wv)
        nbytes = lib.tq_prefill_workspace_bytes(ctypes.byref(g), ctypes.byref(c), ctypes.byref(a))
        ws = (workspace or DecodeWorkspace()).get(nbytes, q.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    _lib.check("tq_prefill_attn", lib.tq_prefill_attn(
        ctypes.byref(g), ctypes.byref(t), ctypes.byref(c), ctypes.byref(a), _stream(q.device)))
    return out


def decode_attention(tables: LayerTables, pages: torch.Tensor, q: torch.Tensor,
                     n_tokens: int, window_k: Optional[torch.Tensor] = None,
                     window_v: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None,
                     workspace: Optional[DecodeWorkspace] = None,
                     num_ctas: int = 0, phases: int = 0,
                     seq_lens: Optional[torch.Tensor] = None,
                     kv_start: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(q K^T * scale) V over the packed tokens [0, n_tokens) of every
    stream plus an optional full-precision window.  q: (B, Hq, 1, D).

    ``phases`` (OR of _lib.PHASE_*) runs a subset of the three kernels; the
    later phases read what the earlier ones left in the same ``workspace``.
    ``seq_lens`` (int32 (B,) on the device) gives each batch row its own
    token count, clamped to [0, n_tokens] (continuous batching).  ``kv_start``
    (int32 (B,) on the device): row b's keys before that position, window
    tokens included, take no weight (left padding)."""
    _require_cuda(pages, q)
    lib = _lib.load()
    if out is None:
        out = torch.empty_like(q)
    g, t, c = tables.geom(), tables.ctables(), _cache_desc(pages)
    keep = []
    a = _decode_args(q, out, n_tokens, window_k, window_v, scale, num_ctas, phases, keep,
                     seq_lens, kv_start)
    nbytes = lib.tq_decode_workspace_bytes(ctypes.byref(g), ctypes.byref(c), ctypes.byref(a))
    if nbytes == 0:
        raise _lib.TqError("tq_decode_workspace_bytes", _lib.TQ_ERR_INVALID, _lib.last_error())
    ws = (workspace or DecodeWorkspace()).get(nbytes, q.device)
    _lib.check("tq_decode_attn", lib.tq_decode_attn(
        ctypes.byref(g), ctypes.byref(t), ctypes.byref(c), ctypes.byref(a),
        ws.data_ptr(), ws.numel(), _stream(q.device)))
    return out


# ---------------------------------------------------------------------------
# Serving operators on a flattened batch of requests
# ---------------------------------------------------------------------------
class _Described:
    """A frozen dataclass of tensors with its C descriptor, made once (2 us) and
    again when a tensor's memory, type or shape is another (``module.to()`` swaps
    them, and may put the new ones at the old address)."""

    def _views(self):
        return [(x.data_ptr(), x.dtype, x.shape, x.stride()) for x in self._tensors()]

    def __post_init__(self):
        object.__setattr__(self, "_c", self._describe())
        object.__setattr__(self, "_of", self._views())

    @property
    def c(self):
        if self._views() != self._of:
            self.__post_init__()
        return self._c


@dataclass(frozen=True, eq=False)
class RopeTable(_Described):
    """Rotary position embedding: row p of ``cos_sin`` (fp32 (positions,
    rot_dim)) holds the cosines, then the sines, of position p's rot_dim / 2
    angles.  Pair i is dims (i, rot_dim / 2 + i) of a head, or (2i, 2i + 1)
    when ``interleaved``; dims from rot_dim on are not rotated.

    ``axes`` (rot_dim / 2 numbers below 4): pair i follows the token's position
    on axis axes[i] (time, height, width of images and video); positions then
    come a row per axis (axis_of_pairs makes the usual orders)."""
    cos_sin: torch.Tensor
    interleaved: bool = False
    axes: Optional[tuple] = None

    def _tensors(self):
        return (self.cos_sin,)

    def _describe(self):
        c = self.cos_sin
        if c.dtype != torch.float32 or c.dim() != 2 or not c.is_contiguous():
            raise ValueError("cos_sin must be a contiguous fp32 (positions, rot_dim) tensor")
        if c.shape[0] < 1 or c.shape[1] < 2 or c.shape[1] % 2:
            raise ValueError(f"cos_sin must hold a position and an even rot_dim, got {tuple(c.shape)}")
        packed = None
        if self.axes is not None:
            pairs = tuple(int(a) for a in self.axes)
            if len(pairs) != c.shape[1] // 2 or len(pairs) > 128 or \
                    not all(0 <= a < 4 for a in pairs):
                raise ValueError(f"axes must give each of the {c.shape[1] // 2} pairs an axis below "
                                 f"4, got {self.axes}")
            packed = (max(pairs) + 1, bytes(pairs))
        object.__setattr__(self, "_axes", packed)
        return _lib.Rope(c.data_ptr(), c.shape[0], c.shape[1], 1 if self.interleaved else 0)

    @property
    def num_axes(self) -> int:
        """Rows of positions that the table's pairs follow (1 without axes)."""
        return 1 if self.axes is None else max(self.axes) + 1

    @staticmethod
    def axis_of_pairs(sections, mixed: bool = False) -> tuple:
        """``axes`` for sections[a] pairs of every axis a: one run of pairs after
        the other, or (``mixed``) one pair of each axis in turn for as long as
        it has any left."""
        left = [int(n) for n in sections]
        if not 1 <= len(left) <= 4 or any(n < 0 for n in left) or not any(left):
            raise ValueError(f"sections must be the pairs of 1 to 4 axes, got {sections}")
        if not mixed:
            return tuple(a for a, n in enumerate(left) for _ in range(n))
        return tuple(a for i in range(max(left)) for a, n in enumerate(left) if i < n)

    @classmethod
    def build(cls, rot_dim: int, positions: int, base: float = 10000.0, interleaved: bool = False,
              inv_freq: Optional[torch.Tensor] = None, scale: float = 1.0,
              device: torch.device = torch.device("cuda"), axes: Optional[tuple] = None) -> "RopeTable":
        """Angles position * base^(-2i / rot_dim), or position * inv_freq[i],
        formed in 64 bits (an fp32 product is off by 0.03 rad at position
        10^6); ``scale`` multiplies the cosines and sines (YaRN's attention
        factor)."""
        if inv_freq is None:
            i = torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device)
            inv_freq = float(base) ** (-i / rot_dim)
        f = inv_freq.to(device=device, dtype=torch.float64)
        if f.shape != (rot_dim // 2,):
            raise ValueError(f"inv_freq must be ({rot_dim // 2},), got {tuple(f.shape)}")
        a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f
        return cls((torch.cat([a.cos(), a.sin()], -1) * scale).float().contiguous(), interleaved,
                   axes)


@dataclass(frozen=True, eq=False)
class HeadNorm(_Described):
    """RMS norm of each head vector: x / sqrt(mean(x^2) + eps) * (weight +
    offset); offset 1 for models that store weight - 1."""
    weight: torch.Tensor
    eps: float = 1e-6
    offset: float = 0.0

    def _tensors(self):
        return (self.weight,)

    def _describe(self):
        w = self.weight
        if w.dim() != 1 or w.dtype not in _DT or not w.is_contiguous():
            raise ValueError("weight must be a contiguous (head_dim,) floating tensor")
        if not self.eps >= 0:
            raise ValueError(f"eps must be >= 0, got {self.eps}")
        return _lib.HeadNorm(w.data_ptr(), _DT[w.dtype], float(self.eps), float(self.offset))


@dataclass(frozen=True, eq=False)
class DiffHeads(_Described):
    """The learned part of differential attention: a pair's result is
    out_scale * norm(A1 V - lam A2 V), A1 and A2 the softmax maps of its two
    query heads.

    ``lam``: fp32 (H,), a pair's own; (N, H), of every row too; or (1,) for all.
    ``keys``: "own", each map has a KV head of its own and V is the values of both
    side by side (2D wide), or "shared", both query heads attend the same KV head.
    ``pairs``: heads of a pair lie next to each other ("adjacent": 2h, 2h + 1) or,
    with own keys, the first ones before the second ones ("halves": h, h + H),
    query heads and KV heads alike.  ``norm``: RMS norm over a pair's result (as
    many weights as it is wide), or None; ``out_scale`` multiplies what is left."""
    lam: torch.Tensor
    keys: str = "own"
    pairs: str = "adjacent"
    norm: Optional[HeadNorm] = None
    out_scale: float = 1.0

    def _tensors(self):
        return (self.lam,)

    def _describe(self):
        x = self.lam
        if x.dtype != torch.float32 or x.dim() not in (1, 2):
            raise ValueError("lam must be an fp32 (H,), (N, H) or (1,) tensor")
        if self.keys not in ("own", "shared"):
            raise ValueError(f"keys must be 'own' or 'shared', got {self.keys!r}")
        if self.pairs not in ("adjacent", "halves"):
            raise ValueError(f"pairs must be 'adjacent' or 'halves', got {self.pairs!r}")
        if self.keys == "shared" and self.pairs != "adjacent":
            raise ValueError("pairs that share their keys lie next to each other ('adjacent')")
        return (x.data_ptr(), 0 if x.dim() == 1 else x.stride(0),
                0 if x.shape[-1] == 1 else x.stride(-1))

    @staticmethod
    def lam_of(q1: torch.Tensor, k1: torch.Tensor, q2: torch.Tensor, k2: torch.Tensor,
               init: float) -> torch.Tensor:
        """lam = exp(q1 . k1) - exp(q2 . k2) + init over the last dim of the learned
        vectors, in 64 bits: (1,) for vectors, (H,) for (H, D).  Computed once, as
        the vectors are fixed in serving."""
        a, b = ((q.double() * k.double()).sum(-1).exp() for q, k in ((q1, k1), (q2, k2)))
        return (a - b + init).float().reshape(-1).detach()


@dataclass(frozen=True, eq=False)
class RowNorm(_Described):
    """Norm of the rows of an activation: (x - mean) / sqrt(mean((x - mean)^2) +
    eps) * (weight + offset) + bias.  mean is 0 (RMS norm) unless ``centered``
    (layer norm); without a weight or a bias that part is left out."""
    weight: Optional[torch.Tensor] = None
    bias: Optional[torch.Tensor] = None
    eps: float = 1e-6
    offset: float = 0.0
    centered: bool = False

    def _tensors(self):
        return tuple(x for x in (self.weight, self.bias) if x is not None)

    def _describe(self):
        for x in self._tensors():
            if x.dim() != 1 or x.dtype not in _DT or not x.is_contiguous():
                raise ValueError("weight and bias must be contiguous (C,) floating tensors")
        w, b = self.weight, self.bias
        if w is not None and b is not None and (w.shape != b.shape or w.dtype != b.dtype):
            raise ValueError("weight and bias differ in shape or type")
        if not self.eps >= 0:
            raise ValueError(f"eps must be >= 0, got {self.eps}")
        one = w if w is not None else b
        return _lib.RowNorm(w.data_ptr() if w is not None else None,
                            b.data_ptr() if b is not None else None,
                            _DT[one.dtype] if one is not None else _lib.TQ_F32, float(self.eps),
                            float(self.offset), 1 if self.centered else 0)


@dataclass(frozen=True, eq=False)
class RaggedBatch(_Described):
    """Requests of different lengths flattened into rows (vLLM's batch): row
    q_start[r] + i is new token i of request r, at position seq_lens[r] -
    (q_start[r + 1] - q_start[r]) + i; seq_lens counts the new tokens.  Both
    stay on the device; ``max_q_len`` (>= the most new tokens of a request)
    shapes launches and never a result.  Rows outside [q_start[0],
    q_start[-1]) belong to no request and are left alone.  Offsets that do not
    ascend within the rows run nothing and set _lib.DEV_BAD_BATCH."""
    q_start: torch.Tensor       # int32 (R + 1,), ascending
    seq_lens: torch.Tensor      # int32 (R,)
    max_q_len: int

    def _tensors(self):
        return (self.q_start, self.seq_lens)

    def _describe(self):
        a, b = self.q_start, self.seq_lens
        if a.dtype != torch.int32 or b.dtype != torch.int32 or a.dim() != 1 or b.dim() != 1 or \
                not a.is_contiguous() or not b.is_contiguous():
            raise ValueError("q_start and seq_lens must be contiguous 1-d int32 tensors")
        if b.shape[0] < 1 or a.shape[0] != b.shape[0] + 1:
            raise ValueError(f"q_start must hold one entry more than seq_lens, got "
                             f"{a.shape[0]} and {b.shape[0]}")
        if a.device != b.device:
            raise ValueError("q_start and seq_lens must be on the same device")
        if self.max_q_len < 0:
            raise ValueError(f"max_q_len must be >= 0, got {self.max_q_len}")
        return _lib.Ragged(b.shape[0], a.data_ptr(), b.data_ptr(), int(self.max_q_len))

    @property
    def requests(self) -> int:
        return self.seq_lens.shape[0]


def _inference_only(name: str, device: torch.device, *ts) -> None:
    """All tensors on ``device`` (CUDA) and none that a backward pass would need
    or that carries a tangent of forward-mode differentiation."""
    grad, forward = torch.is_grad_enabled(), forward_ad._current_level >= 0
    for t in ts:
        if forward and t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no derivative: a tangent would be dropped")
    if device.type != "cuda":
        raise RuntimeError("TurboQuant kernels need CUDA tensors (there is no CPU path)")
    for t in ts:
        if t is None:
            continue
        if t.device != device:
            raise ValueError(f"{name}: tensors on {device} and {t.device}")
        if grad and t.requires_grad:
            raise RuntimeError(f"{name} has no backward pass: call it under torch.no_grad() or "
                               "with detached tensors")


def _on(device: torch.device):
    """The launch's device made current (a no-op when it is)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


class _Descriptors(threading.local):
    """The C descriptors of one call of this thread, packed into one buffer: a
    ctypes structure costs 2 us to fill, more than the kernels of a small step."""

    def __init__(self):
        self.buf = ctypes.create_string_buffer(1408)
        self.base = ctypes.addressof(self.buf)


_desc = _Descriptors()
_T4, _POS, _CACHE = (struct.Struct(f) for f in ("@Pi8q", "@Pi2q", "@PqqPqq"))
_ATTEND = struct.Struct("@PPqPPqfii")
_AXES = struct.Struct("@iq128s")
_NORM_ARGS = struct.Struct("@PPPPPPPfi")
_DIFF = struct.Struct("@PPqPPqfiiiiP2qPf")
# where each descriptor of a call lies in the buffer
_AT_Q, _AT_QO, _AT_K, _AT_KO, _AT_POS, _AT_CACHE, _AT_ARGS = 0, 128, 256, 384, 512, 576, 640
_AT_GATE, _AT_AXES, _AT_DIFF = 896, 1024, 1216
for _s, _c in ((_T4, _lib.Tensor4), (_POS, _lib.Positions), (_CACHE, _lib.Cache),
               (_ATTEND, _lib.AttendArgs), (_NORM_ARGS, _lib.ResidualNormArgs)):
    assert _s.size <= ctypes.sizeof(_c) <= 128
assert _DIFF.size <= ctypes.sizeof(_lib.DiffArgs) <= 192
assert _AXES.size <= ctypes.sizeof(_lib.RopeAxes) <= 192


def _rows(at: int, x: Optional[torch.Tensor], name: str) -> Optional[int]:
    """A flattened (N, H, D) tensor as the (1, H, N, D) view of the C ABI."""
    if x is None:
        return None
    dt = _DT.get(x.dtype)
    if x.dim() != 3:
        raise ValueError(f"{name} must be (rows, heads, head_dim), got shape {tuple(x.shape)}")
    if dt is None:
        raise ValueError(f"unsupported dtype {x.dtype} of {name}")
    n, h, d = x.shape
    sn, sh, sd = x.stride()
    _T4.pack_into(_desc.buf, at, x.data_ptr(), dt, 1, h, n, d, 0, sh, sn, sd)
    return _desc.base + at


def _heads(at: int, x: Optional[torch.Tensor], name: str) -> Optional[int]:
    if x is None or x.dim() != 4:
        return _rows(at, x, name)
    dt = _DT.get(x.dtype)
    if dt is None:
        raise ValueError(f"unsupported dtype {x.dtype} of {name}")
    _T4.pack_into(_desc.buf, at, x.data_ptr(), dt, *x.shape, *x.stride())
    return _desc.base + at


def _positions(pos: Optional[torch.Tensor], b: int, t: int, rope: Optional[RopeTable] = None,
               flat: bool = False):
    """Addresses of the positions' and the axes' descriptors (the latter None
    where one position of a token serves all pairs)."""
    if pos is None:
        return None, None
    if pos.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64, got {pos.dtype}")
    shape, axes = tuple(pos.shape), None
    packed = rope._axes if rope is not None else None
    if shape == (t,):
        stride = (0, pos.stride(0))
    elif packed is not None and shape == ((packed[0], t) if flat else (packed[0], b, t)):
        stride = (0, pos.stride(1)) if flat else pos.stride()[1:]
        _AXES.pack_into(_desc.buf, _AT_AXES, packed[0], pos.stride(0), packed[1])
        axes = _desc.base + _AT_AXES
    elif shape == (b, t):
        stride = pos.stride()
    else:
        each = "" if packed is None else f", with an axis a row ({packed[0]}, " + \
            (f"{t})" if flat else f"{b}, {t})")
        raise ValueError(f"positions must be ({t},) or ({b}, {t}){each}, got {shape}")
    _POS.pack_into(_desc.buf, _AT_POS, pos.data_ptr(), 64 if pos.dtype == torch.int64 else 32,
                   *stride)
    return _desc.base + _AT_POS, axes


def _pages(tables: LayerTables, pages, device: torch.device) -> int:
    paged = isinstance(pages, PagedPages)
    x = pages.pool if paged else pages
    if x.device != device or tables.rot.device != device:
        raise ValueError(f"pages on {x.device}, tables on {tables.rot.device}, heads on {device}")
    if x.dtype != torch.uint8 or x.dim() != (2 if paged else 3) or not x.is_contiguous():
        raise ValueError("pages must be contiguous uint8 (streams, pages, page_bytes), a pool "
                         "(num_blocks, page_bytes)")
    want = page_bytes(tables.head_dim, tables.key_bits, tables.value_bits, tables.qjl)
    if x.shape[-1] != want:
        raise ValueError(f"pages of {x.shape[-1]} bytes where the tables' take {want}")
    if paged:
        bt, pool = pages.block_table, x
        _CACHE.pack_into(_desc.buf, _AT_CACHE, pool.data_ptr(), bt.shape[0], bt.shape[1],
                         bt.data_ptr(), bt.stride(0), pool.shape[0])
    else:
        _CACHE.pack_into(_desc.buf, _AT_CACHE, pages.data_ptr(), pages.shape[0], pages.shape[1],
                         0, 0, 0)
    return _desc.base + _AT_CACHE


def _check_norm(norm: Optional[HeadNorm], d: int) -> None:
    if norm is not None and norm.weight.shape[0] != d:
        raise ValueError(f"a head norm of {norm.weight.shape[0]} weights for heads of {d}")


def _ref(x):
    return None if x is None else ctypes.byref(x)


def _raw_stream(device: torch.device) -> int:
    """The current stream's handle without the Stream object (2 us of 15)."""
    return torch._C._cuda_getCurrentRawStream(
        torch.cuda.current_device() if device.index is None else device.index)


def qk_rope(q: Optional[torch.Tensor], k: Optional[torch.Tensor], rope: Optional[RopeTable],
            positions: Optional[torch.Tensor] = None, q_norm: Optional[HeadNorm] = None,
            k_norm: Optional[HeadNorm] = None, q_out: Optional[torch.Tensor] = None,
            k_out: Optional[torch.Tensor] = None):
    """Norm (optional) and rotation (optional) of query and key heads in one
    pass, in fp32 with one rounding: q (N, Hq, D), k (N, Hkv, D) with
    positions (N,), or q (B, Hq, T, D), k (B, Hkv, T, D) with positions (T,)
    or (B, T); any strides.  A ``rope`` with axes takes positions (axes, N), or
    (axes, B, T), a row for each axis; one position of a token then stands for all
    its axes (text).  Either of q and k may be None.  ``q_out`` /
    ``k_out``: where the results go (may be q / k itself).  A position outside
    the table takes its row 0 and sets _lib.DEV_BAD_POSITION in the device
    status word.  Returns (q_out, k_out)."""
    one = q if q is not None else k
    if one is None:
        raise ValueError("neither q nor k is given")
    if rope is not None and positions is None:
        raise ValueError("a rotation needs positions")
    b, t = (one.shape[0], one.shape[2]) if one.dim() == 4 else (1, one.shape[0])
    _inference_only("qk_rope", one.device, q, k, q_out, k_out, positions,
                    rope.cos_sin if rope is not None else None,
                    q_norm.weight if q_norm is not None else None,
                    k_norm.weight if k_norm is not None else None)
    if q is not None:
        _check_norm(q_norm, q.shape[-1])
        q_out = torch.empty_like(q) if q_out is None else q_out
    if k is not None:
        _check_norm(k_norm, k.shape[-1])
        k_out = torch.empty_like(k) if k_out is None else k_out
    table = rope and rope.c
    pos, axes = _positions(positions, b, t, rope, one.dim() != 4)
    with _on(one.device):
        rest = (_heads(_AT_Q, q, "q"), _heads(_AT_QO, q_out, "q_out"), _ref(q_norm and q_norm.c),
                _heads(_AT_K, k, "k"), _heads(_AT_KO, k_out, "k_out"), _ref(k_norm and k_norm.c),
                _raw_stream(one.device))
        if axes is None:
            _lib.check("tq_qk_rope", _lib.load().tq_qk_rope(_ref(table), pos, *rest))
        else:
            _lib.check("tq_qk_rope_axes",
                       _lib.load().tq_qk_rope_axes(_ref(table), axes, pos, *rest))
    return q_out, k_out


def append_ragged(tables: LayerTables, pages, k: torch.Tensor, v: torch.Tensor,
                  batch: RaggedBatch, rope: Optional[RopeTable] = None,
                  k_norm: Optional[HeadNorm] = None,
                  positions: Optional[torch.Tensor] = None) -> None:
    """Quantise and store a flattened batch's tokens, k and v (N, Hkv, D), at
    their requests' positions; ``pages`` holds stream r * Hkv + h of request
    r, head h.  k is normed and rotated on the way (both optional), by its
    position in its request or by ``positions`` (N,), or (axes, N) where ``rope``
    has axes.  A token whose position
    lies outside the pages is dropped and sets _lib.DEV_BAD_POSITION."""
    _inference_only("append_ragged", k.device, k, v, batch.q_start, positions,
                    rope.cos_sin if rope is not None else None,
                    k_norm.weight if k_norm is not None else None)
    _check_norm(k_norm, k.shape[-1])
    table = rope and rope.c
    pos, axes = _positions(positions, 1, k.shape[0], rope, True)
    with _on(k.device):
        first = (ctypes.byref(tables.geom()), ctypes.byref(tables.ctables()),
                 _pages(tables, pages, k.device),
                 _rows(_AT_K, k, "k"), _rows(_AT_KO, v, "v"), ctypes.byref(batch.c), _ref(table))
        rest = (_ref(k_norm and k_norm.c), pos, _raw_stream(k.device))
        if axes is None:
            _lib.check("tq_append_ragged", _lib.load().tq_append_ragged(*first, *rest))
        else:
            _lib.check("tq_append_ragged_axes",
                       _lib.load().tq_append_ragged_axes(*first, axes, *rest))


def dequantize_ragged(tables: LayerTables, pages, batch: RaggedBatch,
                      k_out: Optional[torch.Tensor], v_out: Optional[torch.Tensor]) -> None:
    """Write the stored keys and values of a flattened batch's tokens into the
    rows of (N, Hkv, D) tensors; either may be None.  A row whose position
    lies outside the pages is zeroed and sets _lib.DEV_BAD_POSITION; rows of no
    request stay as they are.  fp16 and fp32 results are those of fp32
    arithmetic up to its last bits; bf16 ones (head dims 64 and 128) take the
    centroids as fp16, which turns one value in twenty by a step."""
    one = k_out if k_out is not None else v_out
    if one is None:
        raise ValueError("neither k_out nor v_out is given")
    _inference_only("dequantize_ragged", one.device, k_out, v_out, batch.q_start)
    with _on(one.device):
        _lib.check("tq_dequantize_ragged", _lib.load().tq_dequantize_ragged(
            ctypes.byref(tables.geom()), ctypes.byref(tables.ctables()),
            _pages(tables, pages, one.device),
            ctypes.byref(batch.c), _rows(_AT_K, k_out, "k_out"), _rows(_AT_KO, v_out, "v_out"),
            _raw_stream(one.device)))


def attend_ragged(tables: LayerTables, pages, q: torch.Tensor, batch: RaggedBatch,
                  scale: Optional[float] = None, causal: bool = True,
                  out: Optional[torch.Tensor] = None,
                  workspace: Optional[DecodeWorkspace] = None, engine: int = 0) -> torch.Tensor:
    """Attention of a flattened batch q (N, Hq, D) straight off the packed
    pages, each request's rows over its own tokens [0, seq_lens[r]): causal
    (prompt chunks, draft tokens, single tokens, mixed), or with ``causal``
    False every row over all of them (cross attention: the pages hold an
    encoder's states, seq_lens their lengths).  A row that sees no key is zero;
    a request longer than its pages attends what they hold and sets
    _lib.DEV_BAD_POSITION.  Rows of no request stay as they are in ``out``, and
    are not set in an ``out`` of the call's own.

    Work is split along long contexts.  ``engine`` 0 picks the kernels by each
    request's rows and by the type of ``out``, which may differ from q's: bf16
    results come from fp16 operands (relative error 7e-4 beside the rounding's
    1.7e-3), fp16 and fp32 ones from operands of 22 bits (2e-6), whatever the
    size of the values; an fp32 ``out`` is the choice of who wants those bits
    for bf16 queries.  1 is the mma.sync kernel, 2 the tcgen05 kernel (8e-4 in
    any type), 3 the kernel of few query rows.  Pass a ``workspace`` to reuse
    one buffer across calls on one stream."""
    _inference_only("attend_ragged", q.device, q, out, batch.q_start)
    if out is None:
        out = torch.empty_like(q)
    lib = _lib.load()
    g, c, bc = ctypes.byref(tables.geom()), _pages(tables, pages, q.device), batch.c
    _ATTEND.pack_into(_desc.buf, _AT_ARGS, _rows(_AT_Q, q, "q"), _rows(_AT_QO, out, "out"),
                      bc.requests, bc.q_start, bc.seq_lens, bc.max_q_len,
                      scale if scale is not None else 1.0 / math.sqrt(q.shape[-1]),
                      1 if causal else 0, int(engine))
    args = _desc.base + _AT_ARGS
    with _on(q.device):
        nbytes = lib.tq_attend_ragged_workspace_bytes(g, c, args)
        if nbytes == 0:
            raise _lib.TqError("tq_attend_ragged_workspace_bytes", _lib.TQ_ERR_INVALID,
                               _lib.last_error())
        ws = (workspace or DecodeWorkspace()).get(nbytes, q.device)
        _lib.check("tq_attend_ragged", lib.tq_attend_ragged(
            g, ctypes.byref(tables.ctables()), c, args, ws.data_ptr(), ws.numel(),
            _raw_stream(q.device)))
    return out


def diff_attend_ragged(tables: LayerTables, pages, q: torch.Tensor, batch: RaggedBatch,
                       pair: DiffHeads, scale: Optional[float] = None, causal: bool = True,
                       out: Optional[torch.Tensor] = None,
                       workspace: Optional[DecodeWorkspace] = None, engine: int = 0) -> torch.Tensor:
    """Differential attention of a flattened batch straight off the packed pages:
    the query heads q (N, 2H, D) come in pairs (``pair``), each the difference of
    two softmax maps over the request's tokens.  Returns (N, H, 2D) with keys of
    each map's own (the pages hold the KV heads of both maps, values in halves: a
    layer's v of (N, Hkv / 2, 2D) is appended as (N, Hkv, D)), (N, H, D) with
    shared ones.

    Rows, masks, lengths, empty rows, ``scale``, ``causal``, ``engine`` (own keys
    have no tcgen05 kernel: not 2) and ``workspace`` are those of attend_ragged.
    Shared keys, and own keys with codes above 4 bits, leave both maps' results in
    the workspace, 8 bytes an element of the result.  The errors of both maps are
    those of attend_ragged too, and the difference is taken in fp32: where the maps
    nearly cancel, an fp32 ``out`` (operands of 22 bits) keeps what is left."""
    norm = pair.norm
    _inference_only("diff_attend_ragged", q.device, q, out, batch.q_start, pair.lam,
                    norm.weight if norm is not None else None)
    if q.dim() != 3:
        raise ValueError(f"q must be (rows, heads, head_dim), got shape {tuple(q.shape)}")
    own = pair.keys == "own"
    n, h, d = q.shape[0], q.shape[1] // 2, q.shape[2]
    width = 2 * d if own else d
    lam = pair.lam
    if lam.shape[-1] not in (1, h) or (lam.dim() == 2 and lam.shape[0] != n):
        raise ValueError(f"lam must be ({h},), ({n}, {h}) or (1,), got {tuple(lam.shape)}")
    _check_norm(norm, width)
    if out is None:
        out = torch.empty((n, h, width), dtype=q.dtype, device=q.device)
    lib = _lib.load()
    g, c, bc = ctypes.byref(tables.geom()), _pages(tables, pages, q.device), batch.c
    weight = norm.c if norm is not None else None
    _DIFF.pack_into(_desc.buf, _AT_DIFF, _rows(_AT_Q, q, "q"), _rows(_AT_QO, out, "out"),
                    bc.requests, bc.q_start, bc.seq_lens, bc.max_q_len,
                    scale if scale is not None else 1.0 / math.sqrt(d), 1 if causal else 0,
                    int(engine), 0 if own else 1, 1 if pair.pairs == "halves" else 0, *pair.c,
                    ctypes.addressof(weight) if weight is not None else 0, pair.out_scale)
    args = _desc.base + _AT_DIFF
    with _on(q.device):
        nbytes = lib.tq_diff_attend_ragged_workspace_bytes(g, c, args)
        if nbytes == 0:
            raise _lib.TqError("tq_diff_attend_ragged_workspace_bytes", _lib.TQ_ERR_INVALID,
                               _lib.last_error())
        ws = (workspace or DecodeWorkspace()).get(nbytes, q.device)
        _lib.check("tq_diff_attend_ragged", lib.tq_diff_attend_ragged(
            g, ctypes.byref(tables.ctables()), c, args, ws.data_ptr(), ws.numel(),
            _raw_stream(q.device)))
    return out


_GATES = {"none": _lib.GATE_NONE, "sigmoid": _lib.GATE_SIGMOID, "tanh": _lib.GATE_TANH}


def _row_tensor(at: int, x: torch.Tensor, name: str) -> int:
    """A (..., C) tensor of up to four dims as the C ABI's (1, .., rows, C) view."""
    dt = _DT.get(x.dtype)
    if dt is None:
        raise ValueError(f"unsupported dtype {x.dtype} of {name}")
    lead = 4 - x.dim()
    _T4.pack_into(_desc.buf, at, x.data_ptr(), dt, *(1,) * lead, *x.shape, *(0,) * lead, *x.stride())
    return _desc.base + at


def residual_norm(x: torch.Tensor, residual: torch.Tensor, post_norm: Optional[RowNorm] = None,
                  gate: Optional[torch.Tensor] = None, gate_act: str = "none", scale: float = 1.0,
                  pre_norm: Optional[RowNorm] = None, residual_out: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None):
    """A block's output x (..., C) onto the residual stream, and the next block's
    norm of the sum, in one pass:

        y = residual + scale * gate_act(gate) * post_norm(x),   h = pre_norm(y)

    in fp32, y rounded to residual's type and h (formed from the unrounded y) to
    x's.  Norms and gate are optional; ``gate`` broadcasts to x ((C,) a channel's,
    (N, 1) a token's, (N, C)) and goes through ``gate_act``: "none", "sigmoid" or
    "tanh".  x has one to four dims and any strides, C at most 32,768.
    ``residual_out`` / ``out``: where the results go (may be residual / x
    itself).  A row sliced out of a batch gives the bits that the batch gives.
    Returns (residual_out, out); out is None without ``pre_norm``."""
    if x.dim() < 1 or x.dim() > 4 or residual.shape != x.shape:
        raise ValueError(f"x and residual must have one shape of 1 to 4 dims, got "
                         f"{tuple(x.shape)} and {tuple(residual.shape)}")
    if gate_act not in _GATES:
        raise ValueError(f"gate_act must be one of {sorted(_GATES)}, got {gate_act!r}")
    if gate is None and gate_act != "none":
        raise ValueError("gate_act comes with a gate")
    norms = [n for n in (post_norm, pre_norm) if n is not None]
    params = [p for n in norms for p in n._tensors()]
    _inference_only("residual_norm", x.device, x, residual, gate, residual_out, out, *params)
    for p in params:
        if p.shape[0] != x.shape[-1]:
            raise ValueError(f"a norm of {p.shape[0]} values for rows of {x.shape[-1]}")
    if pre_norm is None and out is not None:
        raise ValueError("out comes with pre_norm")
    residual_out = torch.empty_like(residual) if residual_out is None else residual_out
    if pre_norm is not None and out is None:
        out = torch.empty_like(x)
    for name, y in (("residual_out", residual_out), ("out", out)):
        if y is not None and y.shape != x.shape:
            raise ValueError(f"{name} must be {tuple(x.shape)}, got {tuple(y.shape)}")
    if gate is not None:
        gate = torch.broadcast_to(gate, x.shape)
    at_x, at_r = _row_tensor(_AT_Q, x, "x"), _row_tensor(_AT_K, residual, "residual")
    at_g = _row_tensor(_AT_GATE, gate, "gate") if gate is not None else 0
    at_y = _row_tensor(_AT_KO, residual_out, "residual_out")
    at_h = _row_tensor(_AT_QO, out, "out") if out is not None else 0
    post, pre = (n.c if n is not None else None for n in (post_norm, pre_norm))
    _NORM_ARGS.pack_into(_desc.buf, _AT_ARGS, at_x, at_r, at_g, at_y, at_h,
                         ctypes.addressof(post) if post is not None else 0,
                         ctypes.addressof(pre) if pre is not None else 0, scale, _GATES[gate_act])
    with _on(x.device):
        _lib.check("tq_residual_norm", _lib.load().tq_residual_norm(_desc.base + _AT_ARGS,
                                                                    _raw_stream(x.device)))
    return residual_out, out
