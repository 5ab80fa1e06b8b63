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
reported by ``Cache4.check``. There is no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import CoraRuntimeError, InvalidArgument, _check, _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
# Nibble of a 32-bit word that holds column e of its eight (see Weight4).
NIBBLE_OF = (0, 4, 2, 6, 1, 5, 3, 7)


class _CacheArg(C.Structure):
    _fields_ = [("pool", C.c_void_p), ("num_pages", C.c_uint64), ("kv_heads", C.c_uint32),
                ("head_dim", C.c_uint32), ("page_size", C.c_uint32), ("group", C.c_uint32),
                ("status", C.c_void_p)]


class _AppendArg(C.Structure):
    _fields_ = ([(n, C.c_void_p) for n in ("k", "v", "q", "k_out", "v_out", "q_out")]
                + [(n, C.c_int64) for n in ("k_token", "k_head", "v_token", "v_head", "q_token", "q_head")]
                + [(n, C.c_void_p) for n in ("slots", "positions", "rope_cos", "rope_sin")]
                + [("tokens", C.c_uint64), ("rope_rows", C.c_uint64)]
                + [(n, C.c_uint32) for n in ("q_heads", "rotary", "interleaved", "dtype")])


class _AttendArg(C.Structure):
    _fields_ = ([(n, C.c_void_p) for n in ("q", "out", "lse")]
                + [("q_token", C.c_int64), ("q_head", C.c_int64)]
                + [(n, C.c_void_p) for n in ("page_table", "lens", "q_start")]
                + [("table_stride", C.c_int64), ("q_tokens", C.c_uint64), ("workspace_bytes", C.c_uint64),
                   ("workspace", C.c_void_p), ("scale", C.c_float)]
                + [(n, C.c_uint32) for n in ("seqs", "table_width", "q_heads", "max_queries", "window",
                                             "causal", "dtype")])


class _WeightArg(C.Structure):
    _fields_ = [("codes", C.c_void_p), ("meta", C.c_void_p), ("rows", C.c_uint64), ("cols", C.c_uint64),
                ("group", C.c_uint32)]


class _MatvecArg(C.Structure):
    _fields_ = [("x", C.c_void_p), ("bias", C.c_void_p), ("y", C.c_void_p), ("x_stride", C.c_int64),
                ("y_stride", C.c_int64), ("rows", C.c_uint64), ("dtype", C.c_uint32)]


def _bind(L):
    for name, args in (("cora_kv4_append", (C.POINTER(_CacheArg), C.POINTER(_AppendArg), C.c_void_p)),
                       ("cora_kv4_attend", (C.POINTER(_CacheArg), C.POINTER(_AttendArg), C.c_void_p)),
                       ("cora_w4_matvec", (C.POINTER(_WeightArg), C.POINTER(_MatvecArg), C.c_void_p)),
                       ("cora_kv4_status", (C.POINTER(_CacheArg), C.c_void_p))):
        f = getattr(L, name)
        f.restype, f.argtypes = C.c_int, list(args)
    L.cora_kv4_block_bytes.restype, L.cora_kv4_block_bytes.argtypes = C.c_uint64, [C.c_uint32] * 3
    L.cora_kv4_attend_workspace.restype = C.c_uint64
    L.cora_kv4_attend_workspace.argtypes = [C.POINTER(_CacheArg), C.c_uint32, C.c_uint32]


def _need(ok, what):
    if not ok:
        raise InvalidArgument(what)


def _call(f, device, *args):
    """f(*args, stream) on the tensors' device and its current stream."""
    if device.index == torch.cuda.current_device():
        _check(f(*args, torch.cuda.current_stream(device).cuda_stream))
    else:
        with torch.cuda.device(device):
            _check(f(*args, torch.cuda.current_stream(device).cuda_stream))


def _index(t, what, dtype, shape, device):
    _need(t.dtype == dtype and tuple(t.shape) == shape and t.device == device and t.is_contiguous(),
          f"{what} must be a contiguous {dtype} tensor of shape {shape} on {device}")
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
        _bind(_lib)
        _need(head_dim in (64, 128, 256), "head_dim must be 64, 128 or 256")
        _need(group in (64, 128) and group <= head_dim <= 4 * group, "group must be 64 or 128 and at most head_dim")
        _need(16 <= page_size <= 1024 and page_size & (page_size - 1) == 0,
              "page_size must be a power of two from 16 to 1024")
        _need(num_pages >= 1 and kv_heads >= 1, "num_pages and kv_heads must be positive")
        block = int(_lib.cora_kv4_block_bytes(page_size, head_dim, group))
        if pool is None:
            pool = torch.zeros(num_pages, kv_heads, block, dtype=torch.uint8, device=device)
        _need(pool.shape[2] == block, f"a block of this shape has {block} bytes, the pool's have {pool.shape[2]}")
        self.pool, self.device = pool, pool.device
        self.num_pages, self.kv_heads, self.head_dim = num_pages, kv_heads, head_dim
        self.page_size, self.group = page_size, group
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._arg = _CacheArg(pool.data_ptr(), num_pages, kv_heads, head_dim, page_size, group,
                              self.status.data_ptr())
        self._ref = C.byref(self._arg)
        self._work = {}  # attend's workspaces, one per stream (calls on different streams may overlap)

    def _heads(self, x, what, heads=None):
        _need(x.dim() == 3 and x.shape[2] == self.head_dim and (heads is None or x.shape[1] == heads)
              and x.device == self.device and x.stride(2) == 1,
              f"{what} must be (tokens, {heads or 'heads'}, {self.head_dim}) on {self.device}, its last stride 1")
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
        dt = self._heads(k, "k", self.kv_heads)
        T = k.shape[0]
        _need(self._heads(v, "v", self.kv_heads) == dt and v.shape[0] == T, "k and v must be alike")
        a = _AppendArg(k=k.data_ptr(), v=v.data_ptr(), k_token=k.stride(0), k_head=k.stride(1),
                       v_token=v.stride(0), v_head=v.stride(1), tokens=T, dtype=dt,
                       slots=_index(slots, "slots", torch.int64, (T,), self.device))
        qo = ko = vo = None
        if q is not None:
            _need(self._heads(q, "q") == dt and q.shape[0] == T, "q must have k's tokens and type")
            qo = torch.empty(q.shape, dtype=q.dtype, device=self.device)
            a.q, a.q_out, a.q_token, a.q_head, a.q_heads = q.data_ptr(), qo.data_ptr(), q.stride(0), q.stride(1), q.shape[1]
        if rope is not None:
            cos, sin = rope
            _need(positions is not None and cos.dim() == 2, "rope is (cos, sin), each (positions, rotary / 2), and needs positions")
            shape = tuple(cos.shape)
            a.rope_cos = _index(cos, "cos", torch.float32, shape, self.device)
            a.rope_sin = _index(sin, "sin", torch.float32, shape, self.device)
            a.positions = _index(positions, "positions", torch.int32, (T,), self.device)
            a.rope_rows, a.rotary, a.interleaved = shape[0], 2 * shape[1], int(interleaved)
        if values:
            ko = torch.empty(T, self.kv_heads, self.head_dim, dtype=k.dtype, device=self.device)
            vo = torch.empty_like(ko)
            a.k_out, a.v_out = ko.data_ptr(), vo.data_ptr()
        _call(_lib.cora_kv4_append, self.device, self._ref, C.byref(a))
        return Appended(qo, ko, vo)

    def attend(self, q, page_table, lens, q_start=None, max_queries: int = 1, causal=True, window: int = 0,
               scale: Optional[float] = None, return_lse=False, out=None):
        """Softmax attention of new tokens over their sequences' cached ones (their own included).

        q: (rows, heads, head_dim); page_table: int32 (sequences, width), unused entries anything;
        lens: int32 (sequences,) cached tokens. Sequence b asks with rows q_start[b] ..
        q_start[b + 1] - 1 (q_start int32 (sequences + 1,), at most max_queries each; without it
        row b), its last tokens. causal: a token sees those up to itself, with a window only the
        last `window` of them. scale: of the scores, default head_dim ** -0.5. A token that sees
        nothing gets zeros (and lse -inf). Returns out, or (out, lse): lse is fp32 (rows, heads).
        """
        dt = self._heads(q, "q")
        T, Hq, D = q.shape
        _need(page_table.dim() == 2 and page_table.dtype == torch.int32 and page_table.device == self.device
              and page_table.stride(1) == 1, f"page_table must be int32 (sequences, width) on {self.device}")
        B = page_table.shape[0]
        a = _AttendArg(q=q.data_ptr(), q_token=q.stride(0), q_head=q.stride(1), page_table=page_table.data_ptr(),
                       table_stride=page_table.stride(0), table_width=page_table.shape[1],
                       lens=_index(lens, "lens", torch.int32, (B,), self.device), q_tokens=T, q_heads=Hq, seqs=B,
                       scale=D ** -0.5 if scale is None else scale, window=window, causal=int(causal),
                       max_queries=max_queries, dtype=dt)
        _need(window >= 0 and max_queries >= 1, "window and max_queries must not be negative")
        if q_start is not None:
            a.q_start = _index(q_start, "q_start", torch.int32, (B + 1,), self.device)
        else:
            _need(T == B, "q has one row per sequence where q_start is not given")
        if out is None:
            out = torch.empty(T, Hq, D, dtype=q.dtype, device=self.device)
        else:
            _need(out.shape == q.shape and out.dtype == q.dtype and out.device == self.device and out.is_contiguous(),
                  "out must be contiguous, of q's shape and type")
        a.out = out.data_ptr()
        lse = None
        if return_lse:
            lse = torch.empty(T, Hq, dtype=torch.float32, device=self.device)
            a.lse = lse.data_ptr()
        stream = torch.cuda.current_stream(self.device).cuda_stream
        key = (stream, Hq, max_queries)
        work = self._work.get(key) or self._workspace(key)
        a.workspace, a.workspace_bytes = work
        _call(_lib.cora_kv4_attend, self.device, self._ref, C.byref(a))
        return (out, lse) if return_lse else out

    def _workspace(self, key):
        """The stream's workspace, made larger where this shape of call needs more."""
        stream, heads, queries = key
        with torch.cuda.device(self.device):
            size = int(_lib.cora_kv4_attend_workspace(self._ref, heads, queries))
        _need(size > 0, "q_heads must be a multiple of kv_heads")
        buf = self._work.get(stream)
        if buf is None or buf.numel() < size:
            self._work[stream] = buf = torch.zeros(size, dtype=torch.uint8, device=self.device)
            for k in [k for k in self._work if isinstance(k, tuple) and k[0] == stream]:
                del self._work[k]
        self._work[key] = work = (buf.data_ptr(), buf.numel())
        return work

    def check(self):
        """Synchronise the current stream; raise if a call met a bad slot, page, position or row
        range, or if a wait ran out, since the last check."""
        try:
            _call(_lib.cora_kv4_status, self.device, self._ref)
        except CoraRuntimeError:
            self._work.clear()  # a call that gave up may have left its workspace unready
            raise


class Weight4:
    """A (rows, cols) weight matrix in 4 bits: `codes` uint8 (rows, padded / 2) and `meta` fp16
    (rows, padded / group, 2) = (scale, low), padded = cols rounded up to 128. The layout inside
    128 columns is that of the matrix instruction's operands (include/cora_b200.h)."""

    def __init__(self, codes: torch.Tensor, meta: torch.Tensor, cols: int):
        _bind(_lib)
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
        self.device = codes.device
        self._arg = _WeightArg(codes.data_ptr(), meta.data_ptr(), rows, cols, group)
        self._ref = C.byref(self._arg)

    @classmethod
    def quantize(cls, dense: torch.Tensor, group: int = 128) -> "Weight4":
        """Quantise a dense (rows, cols) matrix, as a model is loaded (plain torch, in row blocks)."""
        _need(dense.dim() == 2 and dense.is_cuda and group in (32, 64, 128), "dense must be a CUDA matrix, group 32, 64 or 128")
        rows, cols = dense.shape
        pad = -cols % 128
        step = max(1, (1 << 26) // (cols + pad))
        codes, meta = [], []
        for r in range(0, rows, step):
            x = torch.nn.functional.pad(dense[r:r + step].float(), (0, pad)).unflatten(1, (-1, group))
            low = x.amin(-1, keepdim=True)
            scale = ((x.amax(-1, keepdim=True) - low) / 15.0).clamp(max=65504.0).half().float()
            low = low.clamp(-65504.0, 65504.0).half().float()
            inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
            c = ((x - low) * inv).round().clamp(0, 15).to(torch.int32)
            # 128 columns = 4 j x 4 t x 8 e -> words (t, j), nibbles by e
            c = c.view(x.shape[0], -1, 4, 4, 8).transpose(2, 3)
            word = torch.zeros(c.shape[:-1], dtype=torch.int32, device=dense.device)
            for e, nib in enumerate(NIBBLE_OF):
                word |= c[..., e] << (4 * nib)
            codes.append(word.reshape(x.shape[0], -1).view(torch.uint8))
            meta.append(torch.cat((scale, low), -1).half())
        return cls(torch.cat(codes), torch.cat(meta), cols)


def matvec(x: torch.Tensor, weight: Weight4, bias: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x (..., cols) times the 4-bit weight, plus bias: (..., rows) in x's type. Meant for the few
    rows of decoding (1 to 64); more are correct, 32 rows at a time."""
    _need(x.dim() >= 1 and x.shape[-1] == weight.cols and x.device == weight.device and x.stride(-1) == 1,
          f"x must be (..., {weight.cols}) on {weight.device}, its last stride 1")
    x2 = x if x.dim() == 2 else x.reshape(-1, weight.cols)
    M, N = x2.shape[0], weight.rows
    if bias is not None:
        _need(bias.dtype == x.dtype and tuple(bias.shape) == (N,) and bias.device == x.device and bias.is_contiguous(),
              f"bias must be contiguous ({N},) of x's type")
    if out is None:
        out = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=x.device)
    else:
        _need(tuple(out.shape) == (*x.shape[:-1], N) and out.dtype == x.dtype and out.device == x.device and out.is_contiguous(),
              "out must be contiguous, of x's type, (..., rows)")
    a = _MatvecArg(x2.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), x2.stride(0), N, M,
                   _DTYPES.get(x.dtype, 99))
    _call(_lib.cora_w4_matvec, x.device, weight._ref, C.byref(a))
    return out
