"""Serving operators over a paged key-value cache (include/tarscuda_serve.h), on torch CUDA tensors.

    cache = PagedCache.empty(n_pages, page_size, n_kv, head_dim, batch, max_pages, track=True)
    cache.table[b, :n] = pages                        # the caller hands out the pages
    cache.length.add_(n_new); cache.seen.add_(n_new)  # a step's tokens count before it appends them
    append(cache, k, v, cu)                           # the new rows into the pages
    o = attend_prompt(cache, q, cu, scale)            # the tokens of a prompt, or of a chunk of one
    o = attend(cache, q, scale, weight_out=cache.weight)   # one token per sequence
    evict(cache, budget, sinks=4, recent=256)         # back to the budget by accumulated weight
    token = adjust_logits(logits, history=ids, repetition=r, mask=grammar)

Work is enqueued on torch's current stream of the tensors' device and can be captured into a CUDA
graph. Wrong arguments raise ValueError before anything is enqueued; what only the device can see
(a page id outside the pool, a length beyond the page list) is left out and recorded, and
`device_error` reads it. Only forward passes: the framework trains nothing, and tensors that
require a gradient are refused outside torch.no_grad.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from ._lib import TC_ERR_ARG
from ._lib import lib as _machine_lib

P = ctypes.c_void_p
I32, I64 = ctypes.c_int32, ctypes.c_int64
FP32, BF16, FP16 = 0, 1, 3
DTYPES = {torch.float32: FP32, torch.bfloat16: BF16, torch.float16: FP16}
PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)


class Cache_t(ctypes.Structure):
    _fields_ = [("k", P), ("v", P), ("page_stride", I64), ("slot_stride", I64), ("head_stride", I64),
                ("n_pages", I32), ("page_size", I32), ("n_kv", I32), ("head_dim", I32), ("dtype", I32),
                ("batch", I32), ("max_pages", I32), ("table", P), ("table_stride", I64), ("length", P),
                ("weight", P), ("pos", P), ("track_stride", I64), ("seen", P)]


class Rules_t(ctypes.Structure):
    _fields_ = [("logits", P), ("out", P), ("logits_stride", I64), ("out_stride", I64), ("rows", I32), ("vocab", I32),
                ("history", P), ("history_stride", I64), ("max_history", I32), ("n_history", P), ("n_prompt", P),
                ("repetition", P), ("presence", P), ("frequency", P), ("bias_ids", P), ("bias", P),
                ("bias_stride", I64), ("n_bias", I32), ("mask", P), ("mask_stride", I64), ("token", P), ("none", I32)]


_C, _R = ctypes.POINTER(Cache_t), ctypes.POINTER(Rules_t)
SERVE_SIGNATURES = {
    "tc_kv_append": (ctypes.c_int, [_C, P, P, I32, I64, I64, P, I32, P]),
    "tc_attend": (ctypes.c_int, [_C, P, I64, I64, P, I64, I64, I32, ctypes.c_float, I32, I32, P, P, ctypes.c_uint64,
                                 P]),
    "tc_attend_workspace": (ctypes.c_uint64, [_C, I32, I32]),
    "tc_attend_prompt": (ctypes.c_int, [_C, P, I64, I64, P, I64, I64, I32, P, I32, ctypes.c_float, I32, I32, P,
                                        ctypes.c_uint64, P]),
    "tc_attend_prompt_workspace": (ctypes.c_uint64, [_C, I32, I32, I32, I32]),
    "tc_kv_evict": (ctypes.c_int, [_C, I32, I32, I32, P, P, P, P, ctypes.c_uint64, P]),
    "tc_kv_evict_workspace": (ctypes.c_uint64, [_C, I32]),
    "tc_adjust_logits": (ctypes.c_int, [_R, P]),
}


@functools.lru_cache(None)
def lib():
    L = _machine_lib()
    for name, (res, args) in SERVE_SIGNATURES.items():
        fn = getattr(L, name)
        fn.restype, fn.argtypes = res, args
    return L


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _whole(low: int, **values: int) -> None:
    """Whole numbers from `low` up that the C side holds in 32 bits (ctypes would drop the higher ones)."""
    for name, v in values.items():
        if not low <= v <= 0x7FFFFFFF:
            raise ValueError(f"{name} = {v}: between {low} and 2^31 - 1")


def _check(rc: int, what: str) -> None:
    if rc == TC_ERR_ARG:
        raise ValueError(f"{what}: an argument is out of range, not 16-byte aligned, or shares memory with an output")
    if rc != 0:
        raise RuntimeError(f"{what} failed ({rc})")


def _no_gradient() -> None:
    """Called where a tensor requires a gradient: the calls have no backward pass, and a request for one is
    refused, not silently cut off."""
    if torch.is_grad_enabled():
        raise ValueError("a tensor requires a gradient: the operators have none (detach it, or use torch.no_grad)")


def _ints(t: torch.Tensor, shape: tuple, device: torch.device, name: str) -> None:
    if not (t.dtype is torch.int32 and t.shape == shape and t.device == device and t.is_contiguous()):
        raise ValueError(f"{name}: a contiguous int32 tensor of shape {tuple(shape)} on {device} is wanted")


_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _run(index: int, what: str, fn, *args) -> None:
    """fn(*args, current stream) with device `index` current."""
    if torch.cuda.current_device() == index:
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc:
        _check(rc, what)


def _stride(t: torch.Tensor, d: int) -> int:
    """A dimension's stride; one of a single entry is never stepped over and may be anything."""
    return t.stride(d) if t.shape[d] > 1 else 0


def _apart(t: torch.Tensor) -> bool:
    """Whether the rows of t [.., dim] lie apart in memory, its other dimensions nested in any order."""
    last = t.dim() - 1
    width = t.shape[last]
    for stride, n in sorted((t.stride(d), t.shape[d]) for d in range(last) if t.shape[d] > 1):
        if stride < width:
            return False
        width += stride * (n - 1)
    return True


class PagedCache:
    """Pools, page lists and lengths of `batch` sequences: a handle over the caller's tensors.

    k, v      [n_pages, page_size, n_kv, head_dim] bf16 or fp16, the last dimension contiguous, equal
              strides, no two rows sharing memory (a permuted view of another order is fine; [page,
              kv head, slot, dim] in memory reads fastest)
    table     [batch, max_pages] int32 page ids; entries behind a sequence's length are not read
    length    [batch] int32 slots in use
    weight, pos, seen   what eviction needs, all or none: [batch, n_kv, slots] fp32 attention weight and
              int32 position of each slot (slots >= max_pages * page_size), [batch] int32 tokens taken

    The tensors are fixed for the handle's life; their contents are the caller's to change.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, length: torch.Tensor,
                 weight: torch.Tensor | None = None, pos: torch.Tensor | None = None,
                 seen: torch.Tensor | None = None):
        _need(k.dim() == 4 and k.shape == v.shape and k.stride() == v.stride() and k.dtype == v.dtype and
              k.device == v.device, "k and v: two pools of one shape, type and stride")
        _need(k.dtype in (torch.bfloat16, torch.float16), f"the pools are bf16 or fp16, not {k.dtype}")
        _need(_apart(k), "the pools' rows must lie apart (an expanded dimension shares them)")
        _need(k.is_cuda, "the pools must be on a CUDA device")
        n_pages, page, n_kv, hd = k.shape
        _need(page in PAGE_SIZES, f"page size {page}: one of {PAGE_SIZES}")
        _need(hd in HEAD_DIMS, f"head dim {hd}: one of {HEAD_DIMS}")
        _need(k.stride(3) == 1, "a row's head_dim elements must be contiguous")
        strides = [_stride(k, d) for d in range(3)]
        _need(all(s % 8 == 0 for s in strides) and k.data_ptr() % 16 == 0 and v.data_ptr() % 16 == 0,
              "the pools' rows must be 16-byte aligned")
        _need(table.dim() == 2 and table.dtype == torch.int32 and table.device == k.device and table.shape[0] >= 1
              and table.shape[1] >= 1 and (table.stride(1) == 1 or table.shape[1] == 1) and
              (table.stride(0) >= table.shape[1] or table.shape[0] == 1), "table: int32 [batch, max_pages] on the pools' device")
        batch, max_pages = table.shape
        _ints(length, (batch,), k.device, "length")
        track = [t is not None for t in (weight, pos, seen)]
        _need(all(track) or not any(track), "weight, pos and seen come together")
        if weight is not None:
            _need(weight.dim() == 3 and tuple(weight.shape[:2]) == (batch, n_kv) and
                  weight.shape[2] >= max_pages * page and weight.dtype == torch.float32 and weight.is_contiguous() and
                  weight.device == k.device, "weight: contiguous fp32 [batch, n_kv, slots of the page list]")
            _ints(pos, tuple(weight.shape), k.device, "pos")
            _ints(seen, (batch,), k.device, "seen")
        self._t = (k, v, table, length, weight, pos, seen)
        self.device, self.dtype = k.device, k.dtype
        self.n_pages, self.page_size, self.n_kv, self.head_dim = n_pages, page, n_kv, hd
        self.batch, self.max_pages = batch, max_pages
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.desc = Cache_t(k.data_ptr(), v.data_ptr(), *strides, n_pages, page, n_kv, hd,
                            DTYPES[k.dtype], batch, max_pages, table.data_ptr(), max(_stride(table, 0), max_pages),
                            length.data_ptr(), ptr(weight), ptr(pos), 0 if weight is None else weight.shape[2],
                            ptr(seen))
        self.ref = ctypes.byref(self.desc)
        self.index = k.device.index
        self._sizes: dict = {}                                    # workspace bytes by what asks for them

    def workspace(self, fn, *args) -> tuple:
        """A workspace of its own for one call, from torch's allocator on the current stream: the tensor, its
        address and its size."""
        n = self._sizes.get((fn.__name__, args))
        if n is None:
            if len(self._sizes) >= 1024:
                self._sizes.clear()
            n = self._sizes[fn.__name__, args] = fn(self.ref, *args)
        if n == 0:
            return None, None, 0
        t = torch.empty(n, dtype=torch.uint8, device=self.device)
        return t, t.data_ptr(), n

    k = property(lambda self: self._t[0])
    v = property(lambda self: self._t[1])
    table = property(lambda self: self._t[2])
    length = property(lambda self: self._t[3])
    weight = property(lambda self: self._t[4])
    pos = property(lambda self: self._t[5])
    seen = property(lambda self: self._t[6])

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv: int, head_dim: int, batch: int, max_pages: int,
              dtype: torch.dtype = torch.bfloat16, track: bool = False, device=None) -> "PagedCache":
        """A cache of empty sequences; the pools lie in memory as [page, kv head, slot, dim]."""
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        pool = lambda: torch.empty(n_pages, n_kv, page_size, head_dim, dtype=dtype,  # noqa: E731
                                   device=device).permute(0, 2, 1, 3)
        ints = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)  # noqa: E731
        more = {}
        if track:
            cap = max_pages * page_size
            more = dict(weight=torch.zeros(batch, n_kv, cap, device=device), pos=ints(batch, n_kv, cap), seen=ints(batch))
        return cls(pool(), pool(), ints(batch, max_pages), ints(batch), **more)


def _rows(t: torch.Tensor, cache: PagedCache, heads: int, name: str) -> tuple[int, int, int]:
    """The number of rows of t [rows, heads, head_dim] on the cache's device, its row and head strides."""
    shape, stride = t.shape, t.stride()
    if not (len(shape) == 3 and shape[2] == cache.head_dim and stride[2] == 1 and t.device == cache.device and
            (shape[1] == heads if heads else shape[1] >= 1 and shape[1] % cache.n_kv == 0)):
        raise ValueError(f"{name}: [rows, {heads or 'a multiple of %d' % cache.n_kv} heads, {cache.head_dim}] on "
                         f"{cache.device}, a head's elements contiguous")
    # a dimension of one entry is never stepped over: its stride may be anything
    return shape[0], stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else 0


def _cu(cu: torch.Tensor, cache: PagedCache) -> int:
    _ints(cu, (cache.batch + 1,), cache.device, "cu")
    return cu.data_ptr()


def append(cache: PagedCache, k: torch.Tensor, v: torch.Tensor, cu: torch.Tensor | None = None) -> None:
    """The new tokens' rows [tokens, n_kv, head_dim] (fp32, bf16 or fp16) into the cache, rounded to its
    type. Sequence b owns rows cu[b] .. cu[b+1]-1 (cu None: row b), counted in length and seen already."""
    n, row, head = _rows(k, cache, cache.n_kv, "k")
    code = DTYPES.get(k.dtype)
    if code is None or v.dtype is not k.dtype or v.shape != k.shape or v.stride() != k.stride() or v.device != k.device:
        raise ValueError("k and v: rows of one shape, type (fp32, bf16 or fp16) and stride")
    if cu is None:
        _need(n <= cache.batch, "without cu there is one row per sequence")
    if k.requires_grad or v.requires_grad:
        _no_gradient()
    cu_p = None if cu is None else _cu(cu, cache)
    if n:
        _run(cache.index, "append", lib().tc_kv_append, cache.ref, k.data_ptr(), v.data_ptr(), code, row, head, cu_p, n)


def _attend_args(cache: PagedCache, q: torch.Tensor, out: torch.Tensor | None, window: int, sinks: int) -> tuple:
    """The checked rows of q and out: (rows, out, (q, its strides, out, its strides, heads))."""
    n, row, head = _rows(q, cache, 0, "q")
    if q.dtype is not cache.dtype:
        raise ValueError(f"q has the cache's type {cache.dtype}, not {q.dtype}")
    if not (0 <= window <= 0x7FFFFFFF and 0 <= sinks <= 0x7FFFFFFF):
        _whole(0, window=window, sinks=sinks)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.dtype is not q.dtype or out.shape != q.shape or not (out.is_contiguous() or _apart(out)):
        raise ValueError("out has q's shape and type, its rows apart")
    if q.requires_grad or out.requires_grad:
        _no_gradient()
    _, orow, ohead = _rows(out, cache, q.shape[1], "out")
    return n, out, (q.data_ptr(), row, head, out.data_ptr(), orow, ohead, q.shape[1])


def attend(cache: PagedCache, q: torch.Tensor, scale: float, window: int = 0, sinks: int = 0,
           out: torch.Tensor | None = None, weight_out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one query row per sequence, q [batch, heads, head_dim], over its slots: those of the
    last `window` (0: all) and the first `sinks`. weight_out (cache.weight, or a tensor like it)
    receives cache.weight plus the attention weight each slot draws. Length 0 gives zeros. out must not share
    memory with q."""
    n, out, args = _attend_args(cache, q, out, window, sinks)
    if n != cache.batch:
        raise ValueError(f"{n} query rows for {cache.batch} sequences")
    w = None if weight_out is None else _weight_out(cache, weight_out)
    L = lib()
    ws, ws_p, ws_n = cache.workspace(L.tc_attend_workspace, args[6], int(w is not None))
    _run(cache.index, "attend", L.tc_attend, cache.ref, *args, scale, window, sinks, w, ws_p, ws_n)
    return out


def attend_prompt(cache: PagedCache, q: torch.Tensor, cu: torch.Tensor, scale: float, window: int = 0, sinks: int = 0,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the last tokens of each sequence, rows cu[b] .. cu[b+1]-1 of q [tokens, heads,
    head_dim] for sequence b, each over the slots up to its own position, of the last `window` (0: all)
    and the first `sinks`. Rows at and behind cu[batch] are left alone. out must not share memory with q."""
    n, out, args = _attend_args(cache, q, out, window, sinks)
    cu_p = _cu(cu, cache)
    if n:
        L = lib()
        ws, ws_p, ws_n = cache.workspace(L.tc_attend_prompt_workspace, args[6], n, window, sinks)
        _run(cache.index, "attend_prompt", L.tc_attend_prompt, cache.ref, *args, cu_p, n, scale, window, sinks, ws_p, ws_n)
    return out


def _weight_out(cache: PagedCache, t: torch.Tensor) -> int:
    _need(cache.weight is not None, "the cache keeps no weights")
    if not (t.dtype is torch.float32 and t.shape == cache.weight.shape and t.is_contiguous() and t.device == cache.device):
        raise ValueError("weight_out is laid out as cache.weight")
    return t.data_ptr()


def evict(cache: PagedCache, budget: int, sinks: int = 0, recent: int = 0, length_out: torch.Tensor | None = None,
          weight_out: torch.Tensor | None = None, pos_out: torch.Tensor | None = None) -> None:
    """Cuts every sequence longer than `budget` to it, per key-value head: the first `sinks` and the last
    `recent` positions stay, then the slots of largest weight. Kept slots behind the budget move into
    the holes before it. The new lengths, weights and positions go to the *_out tensors (None: the
    cache's own)."""
    _need(cache.weight is not None, "the cache keeps no weights")
    _whole(1, budget=budget)
    _need(sinks >= 0 and recent >= 0 and sinks + recent <= budget, "0 <= sinks + recent <= budget")
    length_out = cache.length if length_out is None else length_out
    pos_out = cache.pos if pos_out is None else pos_out
    _ints(length_out, (cache.batch,), cache.device, "length_out")
    _ints(pos_out, cache.pos.shape, cache.device, "pos_out")
    w = _weight_out(cache, cache.weight if weight_out is None else weight_out)
    L = lib()
    ws, ws_p, ws_n = cache.workspace(L.tc_kv_evict_workspace, budget)
    _run(cache.index, "evict", L.tc_kv_evict, cache.ref, budget, sinks, recent, length_out.data_ptr(), w,
         pos_out.data_ptr(), ws_p, ws_n)


def _per_row(t: torch.Tensor | None, dtype: torch.dtype, rows: int, device: torch.device, name: str) -> int | None:
    if t is None:
        return None
    if not (t.dtype is dtype and t.shape == (rows,) and t.device == device and t.is_contiguous()):
        raise ValueError(f"{name}: {dtype} [{rows}] on {device}")
    return t.data_ptr()


def _matrix(t: torch.Tensor, dtype: torch.dtype, rows: int, device: torch.device, name: str) -> tuple[int, int, int]:
    """A [rows, n] matrix' pointer, row stride and n; its rows do not overlap."""
    shape, stride = t.shape, t.stride()
    if not (len(shape) == 2 and shape[0] == rows and t.dtype is dtype and t.device == device and
            (stride[1] == 1 or shape[1] <= 1) and (stride[0] >= shape[1] or rows == 1)):
        raise ValueError(f"{name}: {dtype} [{rows}, ..] on {device}, its rows contiguous and apart")
    return t.data_ptr(), stride[0] if rows > 1 else shape[1], shape[1]


def rules_of(logits: torch.Tensor | None, out: torch.Tensor | None = None, history: torch.Tensor | None = None,
             n_history: torch.Tensor | None = None, n_prompt: torch.Tensor | None = None,
             repetition: torch.Tensor | None = None, presence: torch.Tensor | None = None,
             frequency: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
             bias: torch.Tensor | None = None, mask: torch.Tensor | None = None, token: torch.Tensor | None = None,
             none: int = -1, shape: tuple | None = None, device: torch.device | None = None) -> Rules_t:
    """The checked C description of adjust_logits' arguments; without logits, of rules on a decode engine's
    own logits of this shape and device."""
    if not -0x80000000 <= none <= 0x7FFFFFFF:
        _whole(-0x80000000, none=none)
    if logits is None:
        (rows, vocab), dev = shape, device
        x = y = None
        x_stride = y_stride = vocab
    else:
        _need(logits.is_cuda and logits.dim() == 2 and logits.shape[0] >= 1 and logits.shape[1] >= 1,
              "logits: fp32 [rows, vocab] on a CUDA device")
        if logits.requires_grad or (out is not None and out.requires_grad):
            _no_gradient()
        rows, dev = logits.shape[0], logits.device
        x, x_stride, vocab = _matrix(logits, torch.float32, rows, dev, "logits")
        y, y_stride, n = (x, x_stride, vocab) if out is None else _matrix(out, torch.float32, rows, dev, "out")
        _need(n == vocab, "out has the logits' shape")
    h, h_stride, n_h = (None, 0, 0) if history is None else _matrix(history, torch.int32, rows, dev, "history")
    counts = (_per_row(n_history, torch.int32, rows, dev, "n_history"),
              _per_row(n_prompt, torch.int32, rows, dev, "n_prompt"),
              _per_row(repetition, torch.float32, rows, dev, "repetition"),
              _per_row(presence, torch.float32, rows, dev, "presence"),
              _per_row(frequency, torch.float32, rows, dev, "frequency"))
    if n_h == 0:
        _need(history is not None or counts == (None,) * 5, "the penalties need the history")
        h, counts = None, (None,) * 5                             # an empty history has nothing to penalise
    _need((bias is None) == (bias_ids is None), "bias and bias_ids come together")
    ids = val = None
    b_stride = n_b = 0
    if bias is not None:
        ids, b_stride, n_b = _matrix(bias_ids, torch.int32, rows, dev, "bias_ids")
        val, v_stride, n = _matrix(bias, torch.float32, rows, dev, "bias")
        _need(n == n_b and v_stride == b_stride, "bias_ids and bias have one shape and stride")
        if n_b == 0:
            ids = val = None
    m, m_stride = None, 0
    if mask is not None:
        m, m_stride, n = _matrix(mask if mask.dim() == 2 else mask[None], torch.int32, rows if mask.dim() == 2 else 1, dev,
                                 "mask")
        _need(n == (vocab + 31) // 32, f"mask: int32 [rows, {(vocab + 31) // 32}], or one row for all")
        if mask.dim() == 1:
            m_stride = 0
    return Rules_t(x, y, x_stride, y_stride, rows, vocab, h, h_stride, n_h, *counts, ids, val, b_stride, n_b, m, m_stride,
                   _per_row(token, torch.int32, rows, dev, "token"), none)


def adjust_logits(logits: torch.Tensor, token: torch.Tensor | None = None, none: int = -1, **rules) -> torch.Tensor:
    """Penalties, biases and a grammar mask on fp32 logits [rows, vocab], and the greedy pick: the picks
    [rows] int32 (`token`, or a new tensor). Keywords, each optional: out (None: in place; not a shifted
    part of logits), history [rows, ids] int32 with n_history and n_prompt [rows] (prompt ids first),
    repetition / presence / frequency [rows] fp32, bias_ids / bias [rows, entries] (the last entry of a
    token counts), mask int32 words, bit t % 32 of word t // 32 set where token t is allowed. A row
    whose mask allows nothing picks `none`."""
    if token is None:
        token = torch.empty(logits.shape[0], dtype=torch.int32, device=logits.device)
    r = rules_of(logits, token=token, none=none, **rules)
    _run(logits.device.index, "adjust_logits", lib().tc_adjust_logits, ctypes.byref(r))
    return token


def device_error(clear: bool = False) -> int:
    """The first error the current device has recorded (0: none): 51 append, 52 attend, 53
    attend_prompt, 54 evict - a page id outside the pool or a length beyond the page list -, 55 a
    bounded wait of attend_prompt that gave up. Waits for the device."""
    return _machine_lib().tc_wait_error(int(clear))
