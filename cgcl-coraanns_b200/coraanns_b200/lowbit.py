"""A reader in 4 bits beside the index: attention cache and weight products for a language model
that reads what a search retrieved, on the GPU whose memory the index fills (no counterpart in the
reference; ``include/cora_b200.h``, last section, has the formats and the C calls).

    cache = Cache4(num_pages, kv_heads, head_dim)             # paged keys and values, 4 bits
    turned = cache.append(k, v, slots, q=q, rope=(cos, sin), positions=positions)
    out = cache.attend(turned.q, page_table, lens)            # softmax attention over the cache
    w = Weight4.quantize(dense)                               # 4-bit weights, group factors
    y = matvec(out.flatten(1), w)

Tensors are CUDA tensors of torch, bf16 or fp16. Calls enqueue on the current stream of the
tensors' device and return without synchronising; tensors made on another stream have to be ready
on it, as for any torch call. Errors in the arguments raise ``InvalidArgument``; what only the
device can see (a slot, page, position or row range outside its tensor) is skipped there and
reported by ``Cache4.check``. There is no CPU fallback, and there are no gradients: results are
detached from inputs that require them.
"""
from __future__ import annotations

import ctypes as C
import struct
import threading
import weakref
from typing import NamedTuple, Optional

import torch

from . import CoraRuntimeError, InvalidArgument, _check, load_library

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
# Nibble of a 32-bit word that holds column e of its eight (see Weight4).
NIBBLE_OF = (0, 4, 2, 6, 1, 5, 3, 7)


class _CacheArg(C.Structure):
    _fields_ = [("pool", C.c_void_p), ("num_pages", C.c_uint64), ("kv_heads", C.c_uint32),
                ("head_dim", C.c_uint32), ("page_size", C.c_uint32), ("group", C.c_uint32),
                ("status", C.c_void_p)]


class _WeightArg(C.Structure):
    _fields_ = [("codes", C.c_void_p), ("meta", C.c_void_p), ("rows", C.c_uint64), ("cols", C.c_uint64),
                ("group", C.c_uint32)]


# The per-call argument structs, packed in one go (field by field through ctypes costs several
# microseconds a call): cora_kv4_append_args, cora_kv4_attend_args, cora_w4_matvec_args.
_APPEND = struct.Struct("6Q6q4Q2Q4I").pack
_ATTEND = struct.Struct("3Q2q3Qq3Qf7I").pack
_MATVEC = struct.Struct("3Q2qQI4x").pack
_INF = float("inf")
_FLOAT_PAST = 2.0 ** 128 - 2.0 ** 103  # the least that rounds past fp32


def _bind(L):
    ref, args = C.c_void_p, C.c_char_p
    for name, types in (("cora_kv4_append", (ref, args, C.c_void_p)), ("cora_kv4_attend", (ref, args, C.c_void_p)),
                        ("cora_w4_matvec", (ref, args, C.c_void_p)), ("cora_kv4_status", (ref, C.c_void_p))):
        f = getattr(L, name)
        f.restype, f.argtypes = C.c_int, list(types)
    L.cora_kv4_block_bytes.restype, L.cora_kv4_block_bytes.argtypes = C.c_uint64, [C.c_uint32] * 3
    L.cora_kv4_attend_workspace.restype = C.c_uint64
    L.cora_kv4_attend_workspace.argtypes = [ref, C.c_uint32, C.c_uint32]
    return L


_bound = None


def _library():
    global _bound
    if _bound is None:
        _bound = _bind(load_library())
    return _bound


try:  # the current stream's handle without a Stream object around it, the current device
    from torch._C import _cuda_getCurrentRawStream as _stream, _cuda_getDevice as _current_device
except ImportError:
    _current_device = torch.cuda.current_device

    def _stream(index):
        return torch.cuda.current_stream(index).cuda_stream

try:  # whether the current device's current stream is being captured
    from torch._C import _cuda_isCurrentStreamCapturing as _capturing
except ImportError:
    _capturing = torch.cuda.is_current_stream_capturing


class _Workspace:
    """Scratch memory of the attention calls of one stream, which run one after another: all caches
    share it. Never part of a captured graph."""
    __slots__ = ("held", "__weakref__")

    def __init__(self):
        self.held = (0, 0, None)  # address, bytes, the tensor: replaced as a whole


_workspaces = weakref.WeakValueDictionary()  # (device, stream handle) -> _Workspace, alive while a cache uses it
_workspaces_lock = threading.Lock()


def _refuse(what):
    raise InvalidArgument(what)


def _need(ok, what):
    if not ok:
        raise InvalidArgument(what)


def _call(f, index, *args):
    """f(*args, stream) on device `index` and its current stream."""
    if index == _current_device():
        rc = f(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _stream(index))
    if rc:
        _check(rc)


def _index(t, what, dtype, shape, device):
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device.index or not t.is_contiguous():
        _refuse(f"{what} must be a contiguous {dtype} tensor of shape {shape} on {device}")
    return t.data_ptr()


class Appended(NamedTuple):
    """What Cache4.append gives back: the rotated queries, and (values=True) what the stored codes
    stand for."""
    q: Optional[torch.Tensor]
    k: Optional[torch.Tensor]
    v: Optional[torch.Tensor]


class Cache4:
    """Keys and values of many sequences in pages, 4 bits each with two fp16 factors per group.

    head_dim 64, 128 or 256; group 64 or 128 consecutive dimensions (default: the smaller of 128
    and head_dim); page_size a power of two from 16 to 1024 tokens. ``pool`` is the cache itself,
    uint8 (num_pages, kv_heads, bytes of a block); who owns which page is the caller's page table.
    One cache may be used on several streams; calls that touch the same pages are the caller's to
    order.
    """

    def __init__(self, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64,
                 group: Optional[int] = None, device="cuda"):
        group = min(128, head_dim) if group is None else group
        self._setup(None, num_pages, kv_heads, head_dim, page_size, group, torch.device(device))

    @classmethod
    def from_pool(cls, pool: torch.Tensor, page_size: int, head_dim: int, group: Optional[int] = None):
        """A cache over an existing pool (e.g. one restored from a checkpoint)."""
        _need(pool.dtype == torch.uint8 and pool.dim() == 3 and pool.is_contiguous() and pool.is_cuda,
              "pool must be a contiguous CUDA uint8 tensor (pages, kv_heads, block bytes)")
        self = cls.__new__(cls)
        group = min(128, head_dim) if group is None else group
        self._setup(pool, pool.shape[0], pool.shape[1], head_dim, page_size, group, pool.device)
        return self

    def _setup(self, pool, num_pages, kv_heads, head_dim, page_size, group, device):
        self._lib = _library()
        _need(head_dim in (64, 128, 256), "head_dim must be 64, 128 or 256")
        _need(group in (64, 128) and group <= head_dim <= 4 * group, "group must be 64 or 128 and at most head_dim")
        _need(16 <= page_size <= 1024 and page_size & (page_size - 1) == 0,
              "page_size must be a power of two from 16 to 1024")
        _need(num_pages >= 1 and kv_heads >= 1, "num_pages and kv_heads must be positive")
        block = int(self._lib.cora_kv4_block_bytes(page_size, head_dim, group))
        if pool is None:
            pool = torch.zeros(num_pages, kv_heads, block, dtype=torch.uint8, device=device)
        _need(pool.shape[2] == block, f"a block of this shape has {block} bytes, the pool's have {pool.shape[2]}")
        self.pool, self.device = pool, pool.device
        self.num_pages, self.kv_heads, self.head_dim = num_pages, kv_heads, head_dim
        self.page_size, self.group = page_size, group
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._arg = _CacheArg(pool.data_ptr(), num_pages, kv_heads, head_dim, page_size, group,
                              self.status.data_ptr())
        self._ref = C.addressof(self._arg)
        self._dev = self.device.index
        self._spaces = {}  # stream handle -> _Workspace (calls on different streams may overlap)
        self._bytes = {}   # bits of the rows per key head -> bytes of a workspace

    def _heads(self, x, what, shape):
        """The type code of a (tokens, heads, head_dim) tensor."""
        if x.shape != shape or x.get_device() != self._dev or x.stride(2) != 1:
            _refuse(f"{what} must be {shape} on {self.device}, its last stride 1")
        return _DTYPES.get(x.dtype, 99)

    def append(self, k, v, slots, q=None, rope=None, positions=None, interleaved=False, values=False) -> Appended:
        """Quantise and store keys and values of new tokens; rotate keys and queries first.

        k, v: (tokens, kv_heads, head_dim), any strides but the last; slots: int64 (tokens,),
        page * page_size + offset, negative to store nothing. rope: (cos, sin), fp32
        (positions, rotary / 2), and positions: int32 (tokens,), its rows; rotated are the first
        `rotary` dimensions in pairs (i, i + rotary / 2), or (2i, 2i + 1) when interleaved. q:
        (tokens, heads, head_dim), returned rotated. values: also return the keys and values that
        the stored codes stand for, as k and v of the result. A slot may appear once.
        """
        D, dev = self.head_dim, self.device
        if k.dim() != 3:
            _refuse(f"k must be (tokens, {self.kv_heads}, {D})")
        T = k.shape[0]
        shape = (T, self.kv_heads, D)
        dt = self._heads(k, "k", shape)
        if self._heads(v, "v", shape) != dt:
            _refuse("k and v must be of one type")
        qo = ko = vo = None
        qp = qop = kop = vop = qt = qh = heads = pos = cosp = sinp = rows = rotary = 0
        if q is not None:
            if q.dim() != 3 or self._heads(q, "q", (T, q.shape[1], D)) != dt:
                _refuse("q must be (tokens, heads, head_dim) of k's type")
            heads = q.shape[1]
            qo = torch.empty((T, heads, D), dtype=q.dtype, device=dev)
            qp, qop, (qt, qh, _) = q.data_ptr(), qo.data_ptr(), q.stride()
        if rope is not None:
            cos, sin = rope
            if positions is None or cos.dim() != 2:
                _refuse("rope is (cos, sin), each (positions, rotary / 2), and needs positions")
            rows, rotary = cos.shape
            cosp = _index(cos, "cos", torch.float32, cos.shape, dev)
            sinp = _index(sin, "sin", torch.float32, cos.shape, dev)
            pos = _index(positions, "positions", torch.int32, (T,), dev)
        if values:
            ko, vo = torch.empty(shape, dtype=k.dtype, device=dev), torch.empty(shape, dtype=k.dtype, device=dev)
            kop, vop = ko.data_ptr(), vo.data_ptr()
        kt, kh, _ = k.stride()
        vt, vh, _ = v.stride()
        _call(self._lib.cora_kv4_append, self._dev, self._ref, _APPEND(
            k.data_ptr(), v.data_ptr(), qp, kop, vop, qop, kt, kh, vt, vh, qt, qh,
            _index(slots, "slots", torch.int64, (T,), dev), pos, cosp, sinp, T, rows, heads, 2 * rotary, bool(interleaved), dt))
        return Appended(qo, ko, vo)

    def attend(self, q, page_table, lens, q_start=None, max_queries: int = 1, causal=True, window: int = 0,
               scale: Optional[float] = None, return_lse=False, out=None):
        """Softmax attention of new tokens over their sequences' cached ones (their own included).

        q: (rows, heads, head_dim); page_table: int32 (sequences, width), unused entries anything;
        lens: int32 (sequences,) cached tokens. Sequence b asks with rows q_start[b] ..
        q_start[b + 1] - 1 (q_start int32 (sequences + 1,), at most max_queries each; without it
        row b), its last tokens. causal: a token sees those up to itself, with a window only the
        last `window` of them. scale: of the scores, default head_dim ** -0.5. A token that sees
        nothing gets zeros (and lse -inf), as do rows of q outside all ranges. Returns out, or (out, lse): lse is fp32 (rows, heads). out
        may be q itself (a row is written once all that read it have), else it must not overlap q.
        """
        if self._dev != _current_device():
            with torch.cuda.device(self._dev):
                return self.attend(q, page_table, lens, q_start, max_queries, causal, window, scale, return_lse, out)
        dev = self.device
        if q.dim() != 3 or page_table.dim() != 2:
            _refuse("q must be (rows, heads, head_dim), page_table (sequences, width)")
        T, Hq, D = shape = q.shape
        dt = self._heads(q, "q", (T, Hq, self.head_dim))
        B, width = page_table.shape
        stride, last = page_table.stride()
        if page_table.dtype is not torch.int32 or page_table.get_device() != self._dev or (last != 1 and width > 1):
            _refuse(f"page_table must be int32 (sequences, width) on {dev}")
        if not 0 <= window <= 0x7fffffff or not 1 <= max_queries <= 0xffffffff:
            _refuse("window must fit an int and not be negative, max_queries must be positive and fit 32 bits")
        if scale is None:
            scale = D ** -0.5
        elif _FLOAT_PAST <= abs(scale) < _INF:
            _refuse("scale must fit fp32")
        qs = 0
        if q_start is not None:
            qs = _index(q_start, "q_start", torch.int32, (B + 1,), dev)
        elif T != B:
            _refuse("q has one row per sequence where q_start is not given")
        if out is None:
            out = torch.empty(shape, dtype=q.dtype, device=dev)
        elif out.shape != shape or out.dtype != q.dtype or out.device != dev or not out.is_contiguous():
            _refuse("out must be contiguous, of q's shape and type")
        lse, lp = None, 0
        if return_lse:
            lse = torch.empty((T, Hq), dtype=torch.float32, device=dev)
            lp = lse.data_ptr()
        stream = _stream(self._dev)
        bits = (max_queries * (Hq // self.kv_heads) - 1).bit_length()  # of the rows per key head
        space, size = self._spaces.get(stream), self._bytes.get(bits)
        held = (0, 0, None) if space is None or size is None else space.held  # (kept until the call is enqueued)
        if not held[1] or held[1] < size or _capturing():
            held = self._workspace(bits, stream)
        work, size, _ = held
        qt, qh, _ = q.stride()
        rc = self._lib.cora_kv4_attend(self._ref, _ATTEND(
            q.data_ptr(), out.data_ptr(), lp, qt, qh, page_table.data_ptr(),
            _index(lens, "lens", torch.int32, (B,), dev), qs, stride, T, size, work,
            scale, B, width, Hq, max_queries, window, bool(causal), dt), stream)
        if rc:
            _check(rc)
        return (out, lse) if return_lse else out

    def _workspace(self, bits, stream):
        """(address, bytes, tensor) for a call of up to 2^bits rows per key head on the current stream."""
        size = self._bytes.get(bits)
        if size is None:
            size = int(self._lib.cora_kv4_attend_workspace(self._ref, self.kv_heads, min(1 << bits, 0xffffffff)))
            if not size:
                raise CoraRuntimeError(load_library().cora_last_error().decode())
            self._bytes[bits] = size
        if _capturing():
            # A graph's own: its replays may overlap calls, and other graphs, of this stream, and outlive
            # what is kept here. The call itself adds the node that readies it.
            buf = torch.empty(size, dtype=torch.uint8, device=self.device)
            return buf.data_ptr(), size, buf
        dev = self._dev
        with _workspaces_lock:
            space = _workspaces.get((dev, stream))
            if space is None:
                _workspaces[dev, stream] = space = _Workspace()
            if space.held[1] < size:
                buf = torch.zeros(size, dtype=torch.uint8, device=self.device)
                space.held = (buf.data_ptr(), size, buf)
            self._spaces[stream] = space
            return space.held

    def check(self):
        """Synchronise the current stream; raise if a call met a bad slot, page, position or row
        range, or if a wait ran out, since the last check. Calls on other streams are covered where
        they are ordered before this one."""
        try:
            _call(self._lib.cora_kv4_status, self._dev, self._ref)
        except CoraRuntimeError:
            # a call that gave up may have left a workspace unready: the next ones take fresh memory
            with _workspaces_lock:
                for (dev, _), space in list(_workspaces.items()):
                    if dev == self._dev:
                        space.held = (0, 0, None)
            raise


class Weight4:
    """A (rows, cols) weight matrix in 4 bits: `codes` uint8 (rows, padded / 2) and `meta` fp16
    (rows, padded / group, 2) = (scale, low), padded = cols rounded up to 128. The layout inside
    128 columns is that of the matrix instruction's operands (include/cora_b200.h)."""

    def __init__(self, codes: torch.Tensor, meta: torch.Tensor, cols: int):
        self._lib = _library()
        padded = -(-cols // 128) * 128
        _need(codes.dtype == torch.uint8 and codes.dim() == 2 and codes.is_contiguous() and codes.is_cuda
              and codes.shape[1] * 2 == padded, f"codes must be contiguous CUDA uint8 (rows, {padded // 2})")
        rows = codes.shape[0]
        _need(meta.dtype == torch.float16 and meta.dim() == 2 + (meta.dim() == 3) and meta.is_contiguous()
              and meta.device == codes.device and meta.shape[0] == rows, "meta must be contiguous fp16 (rows, groups, 2)")
        groups = meta.shape[1] if meta.dim() == 3 else meta.shape[1] // 2
        group = padded // max(1, groups)
        _need(groups * group == padded and group in (32, 64, 128) and meta.numel() == rows * groups * 2,
              "meta must hold a pair for each group of 32, 64 or 128 columns")
        self.codes, self.meta, self.rows, self.cols, self.group = codes, meta, rows, cols, group
        self.device, self._dev = codes.device, codes.device.index
        self._arg = _WeightArg(codes.data_ptr(), meta.data_ptr(), rows, cols, group)
        self._ref = C.addressof(self._arg)

    @classmethod
    def quantize(cls, dense: torch.Tensor, group: int = 128) -> "Weight4":
        """Quantise a dense (rows, cols) matrix, as a model is loaded (plain torch, in row blocks)."""
        _need(dense.dim() == 2 and dense.is_cuda and group in (32, 64, 128), "dense must be a CUDA matrix, group 32, 64 or 128")
        rows, cols = dense.shape
        _need(cols >= 1, "dense must have columns")
        pad = -cols % 128
        step = max(1, (1 << 26) // (cols + pad))
        codes, meta = [], []
        for r in range(0, max(1, rows), step):
            x = torch.nn.functional.pad(dense[r:r + step].float(), (0, pad)).unflatten(1, (-1, group))
            low = x.amin(-1, keepdim=True)
            scale = ((x.amax(-1, keepdim=True) - low) * (1 / 15)).clamp(max=65504.0).half().float()
            low = low.clamp(-65504.0, 65504.0).half().float()
            inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
            c = ((x - low) * inv).round().clamp(0, 15).to(torch.int32)
            # 128 columns = 4 j x 4 t x 8 e -> words (t, j), nibbles by e
            c = c.view(x.shape[0], (cols + pad) // 128, 4, 4, 8).transpose(2, 3)
            word = torch.zeros(c.shape[:-1], dtype=torch.int32, device=dense.device)
            for e, nib in enumerate(NIBBLE_OF):
                word |= c[..., e] << (4 * nib)
            codes.append(word.reshape(x.shape[0], (cols + pad) // 8).view(torch.uint8))
            meta.append(torch.cat((scale, low), -1).half())
        return cls(torch.cat(codes), torch.cat(meta), cols)


def matvec(x: torch.Tensor, weight: Weight4, bias: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x (..., cols) times the 4-bit weight, plus bias: (..., rows) in x's type. Meant for the few
    rows of decoding (1 to 64); more are correct, 32 rows at a time. out must not overlap x."""
    dev, N, dims = weight.device, weight.rows, x.dim()
    if not dims or x.shape[-1] != weight.cols or x.get_device() != weight._dev or (x.stride(-1) != 1 and weight.cols > 1):
        _refuse(f"x must be (..., {weight.cols}) on {dev}, its last stride 1")
    x2 = x if dims == 2 else x.reshape(-1, weight.cols)
    M = x2.shape[0]
    shape = (M, N) if dims == 2 else (*x.shape[:-1], N)
    bp = 0
    if bias is not None:
        bp = _index(bias, "bias", x.dtype, (N,), dev)
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=dev)
    elif out.shape != shape or out.dtype != x.dtype or out.device != dev or not out.is_contiguous():
        _refuse("out must be contiguous, of x's type, (..., rows)")
    elif M and N:  # (blocks read x while others write)
        first, end = x2.data_ptr(), x2.data_ptr() + 2 * ((M - 1) * x2.stride(0) + weight.cols)
        if out.data_ptr() < end and first < out.data_ptr() + 2 * M * N:
            _refuse("out must not overlap x")
    _call(weight._lib.cora_w4_matvec, weight._dev, weight._ref, _MATVEC(
        x2.data_ptr(), bp, out.data_ptr(), x2.stride(0), N, M, _DTYPES.get(x.dtype, 99)))
    return out
