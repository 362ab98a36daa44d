"""A text decoder's operators (include/ocrhip.h): a paged cache of keys and values, attention over
prompts and of single tokens over the cache, beam search.

Arrays are device memory: torch tensors on the context's device, or DeviceArray over a
DeviceBuffer. A head's values, and the heads of a token, lie one after another; tokens may lie
further apart. Every call is queued on the context's stream and returns at once; Context.acquire
and Context.release order it with other streams. The memory must outlive the work.
"""
from __future__ import annotations

import ctypes
import sys
import warnings

P, U32, I32, I64, F32, F64 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_double
_TYPES = {"float32": 0, "float16": 1, "bfloat16": 2, "int8": 3, "uint8": 4, "float8_e4m3fn": 4, "int32": 5}
_SHORT = {"f32": 0, "f16": 1, "bf16": 2, "i8": 3, "e4m3": 4, "i32": 5}
_NAMES = {v: k for k, v in _SHORT.items()}
_SIZES = {0: 4, 1: 2, 2: 2, 3: 1, 4: 1, 5: 4}
_known = {}  # a dtype object's code


class ocr_kv_cache(ctypes.Structure):
    _fields_ = [("k", P), ("v", P), ("k_scale", P), ("v_scale", P), ("pages", U32), ("heads", U32), ("page", U32), ("dim", U32),
                ("type", I32)]


class ocr_page_table(ctypes.Structure):
    _fields_ = [("table", P), ("rows", U32), ("width", U32)]


class ocr_kv_append_args(ctypes.Structure):
    _fields_ = [("seq", P), ("pos", P), ("qkv", P), ("type", I32), ("n", U32), ("q_heads", U32), ("stride", I64), ("q_norm", P),
                ("k_norm", P), ("eps", F32), ("rot", U32), ("theta", F64), ("adjacent", I32), ("q", P), ("k", P), ("out_type", I32)]


class ocr_attention_args(ctypes.Structure):
    _fields_ = [("q", P), ("k", P), ("v", P), ("out", P), ("type", I32), ("n", U32), ("q_heads", U32), ("kv_heads", U32), ("dim", U32),
                ("q_stride", I64), ("k_stride", I64), ("v_stride", I64), ("out_stride", I64), ("docs", P), ("ndocs", U32),
                ("prefix", P), ("scale", F32), ("cap", F32), ("slopes", P)]


class ocr_decode_args(ctypes.Structure):
    _fields_ = [("lens", P), ("q", P), ("out", P), ("type", I32), ("q_heads", U32), ("q_stride", I64), ("out_stride", I64),
                ("scale", F32), ("cap", F32), ("slopes", P)]


class ocr_beam_args(ctypes.Structure):
    _fields_ = [("logits", P), ("type", I32), ("groups", U32), ("beams", U32), ("vocab", U32), ("stride", I64), ("scores", P),
                ("finished", P), ("eos", I32), ("out_scores", P), ("parents", P), ("tokens", P), ("out_finished", P)]


class DeviceArray:
    """A DeviceBuffer's memory as an array: shape, a type of "f32", "f16", "bf16", "i8", "e4m3" or
    "i32", and strides in values (the last dimensions' by default)."""

    def __init__(self, buffer, shape, dtype: str, strides=None):
        if dtype not in _SHORT:
            raise _error(f"a type of {sorted(_SHORT)} is wanted, not {dtype!r}")
        self.buffer, self.shape, self.dtype = buffer, tuple(int(v) for v in shape), dtype
        if strides is None:
            strides, n = [], 1
            for v in reversed(self.shape):
                strides.insert(0, n)
                n *= v
        self.strides = tuple(int(v) for v in strides)
        if len(self.strides) != len(self.shape) or min(self.shape + self.strides, default=0) < 0:
            raise _error(f"shape {self.shape} with strides {self.strides}")
        last = sum((n - 1) * s for n, s in zip(self.shape, self.strides)) + 1 if 0 not in self.shape else 0
        if last * _SIZES[_SHORT[dtype]] > buffer.nbytes:
            raise _error(f"an array of shape {self.shape} does not fit a buffer of {buffer.nbytes} bytes")

    def data_ptr(self):
        return self.buffer.ptr

    def stride(self):
        return self.strides


def _root():
    return sys.modules[__package__]


def _error(message):
    return _root().OcrError(message)


def _call(name, *args):
    root = _root()
    if getattr(root.lib(), name)(*args) != 0:
        raise root.OcrError(root.lib().ocr_last_error().decode())


_tensors = None  # the module, False where it is not there


def _native(name, ctx, *args):
    """The call on torch tensors by ocrhip._tensors; False if that leaves it to the checks here, which
    say what is wrong or take arrays of another kind. Without the module they do all of it, a few
    microseconds a call slower."""
    global _tensors
    if not _tensors:
        if _tensors is False or "torch" not in sys.modules:
            return False
        try:
            from . import _tensors as module
        except ImportError as e:
            warnings.warn(f"ocrhip._tensors is not there (python -m ocrhip.build makes it); calls on tensors are checked in Python: {e}",
                          RuntimeWarning, stacklevel=3)
            _tensors = False
            return False
        lib = _root().lib()
        module.bind(*[ctypes.cast(getattr(lib, f"ocr_{f}_device"), ctypes.c_void_p).value
                      for f in ("kv_append", "kv_read", "attention", "decode_attention", "beam_select", "kv_fork")])
        _tensors = module
    rc = getattr(_tensors, name)(ctx.handle, ctx.device, *args)
    if rc > 0 or rc == -1:
        raise _error(_root().lib().ocr_last_error().decode())
    return rc == 0


def _code(x, what):
    code = _known.get(x.dtype)
    if code is None:
        d = x.dtype
        code = _SHORT.get(d) if isinstance(d, str) else _TYPES.get(str(d).replace("torch.", ""))
        if code is None:
            raise _error(f"{what}: arrays of {d} are not taken")
        _known[d] = code
    return code


def _device(ctx, x, what):
    """Refuses what is not in the memory of the context's device."""
    try:
        if isinstance(x, DeviceArray):
            there = x.buffer.ctx.device == ctx.device and bool(x.buffer.ptr)
        else:
            d = x.device
            there = d.type == "cuda" and d.index == ctx.device
    except AttributeError:
        there = False
    if not there:
        raise _error(f"{what} is not an array in the memory of device {ctx.device}")


def _array(ctx, x, what, types, shape):
    """The address of x, an array of one of `types` and exactly this shape, its values one after
    another; None stays None."""
    if x is None:
        return None
    _device(ctx, x, what)
    if _code(x, what) not in types:
        raise _error(f"{what}: {' or '.join(_NAMES[t] for t in types)} is wanted, not {x.dtype}")
    if tuple(x.shape) != shape:
        raise _error(f"{what}: shape {shape} is wanted, not {tuple(x.shape)}")
    want = 1
    for n, s in zip(reversed(shape), reversed(x.stride())):
        if n != 1 and s != want and 0 not in shape:
            raise _error(f"{what}: its values do not lie one after another")
        want *= n
    return x.data_ptr() or None


def _tokens(ctx, x, what, types, n=None, heads=None, dim=None):
    """(address, tokens, heads, dim, stride) of x [tokens][heads][dim], whose tokens may lie apart."""
    _device(ctx, x, what)
    if _code(x, what) not in types:
        raise _error(f"{what}: {' or '.join(_NAMES[t] for t in types)} is wanted, not {x.dtype}")
    shape, strides = x.shape, x.stride()
    if len(shape) != 3 or any(w is not None and w != v for w, v in zip((n, heads, dim), shape)):
        want = tuple("any" if v is None else v for v in (n, heads, dim))
        raise _error(f"{what}: shape {want} is wanted, not {tuple(shape)}")
    n, heads, dim = shape
    if n and ((dim > 1 and strides[2] != 1) or (heads > 1 and strides[1] != dim)):
        raise _error(f"{what}: a token's values do not lie one after another")
    row = heads * dim
    return x.data_ptr() or None, n, heads, dim, strides[0] if n > 1 else row


_I32, _F32, _F16, _ANY = (5,), (0,), (1, 2), (0, 1, 2)
_PAIRS = {"halves": False, "adjacent": True}


class KvCache:
    """A paged cache: a pool of pages of `page` positions that hold heads x dim keys and values of
    type "f16", "bf16", "i8" or "e4m3" (ocr_kv_cache). Which pages a sequence has is in the tables
    [sequences][entries] (int32) that the calls take. memory: the caller's (k, v, k_scale,
    v_scale), [pages][heads][page][dim] and [pages][heads][page] float32 (None for the 16-bit
    types); without it the cache allocates its own."""

    def __init__(self, ctx, pages: int, page: int, heads: int, dim: int, dtype: str = "i8", memory=None):
        if dtype not in ("f16", "bf16", "i8", "e4m3"):
            raise _error(f"cache: f16, bf16, i8 or e4m3 is wanted, not {dtype!r}")
        if min(pages, page, heads, dim) < 1:
            raise _error("cache: empty")
        if max(pages, page, heads, dim) >= 2 ** 32:  # ctypes would cut them
            raise _error(f"cache: sizes {(pages, page, heads, dim)} are past 32 bits")
        self.ctx, self.pages, self.page, self.heads, self.dim, self.dtype = ctx, pages, page, heads, dim, dtype
        code = _SHORT[dtype]
        shape = (pages, heads, page, dim)
        if memory is None:
            count = pages * heads * page
            k, v = (DeviceArray(ctx.alloc(count * dim * _SIZES[code]), shape, dtype) for _ in range(2))
            ks = vs = None
            if code >= 3:
                ks, vs = (DeviceArray(ctx.alloc(count * 4), shape[:3], "f32") for _ in range(2))
            memory = (k, v, ks, vs)
        self.k, self.v, self.k_scale, self.v_scale = memory
        scales = [_array(ctx, x, "cache scales", _F32, shape[:3]) for x in memory[2:]] if code >= 3 else [None, None]
        if code >= 3 and None in scales:
            raise _error("cache: an 8-bit cache needs scales")
        self._c = ocr_kv_cache(_array(ctx, self.k, "cache keys", (code,), shape), _array(ctx, self.v, "cache values", (code,), shape),
                               *scales, pages, heads, page, dim, code)
        self._at = ctypes.addressof(self._c)

    def _table(self, table):
        if len(table.shape) != 2:
            raise _error(f"page table: shape [sequences][entries] is wanted, not {tuple(table.shape)}")
        rows, width = table.shape
        return ocr_page_table(_array(self.ctx, table, "page table", _I32, (rows, width)), rows, width)

    def append(self, table, seq, pos, qkv, q, k=None, q_norm=None, k_norm=None, eps: float = 1e-6, rot: int | None = None,
               theta: float = 1e4, pairs: str = "halves"):
        """Projections qkv [n][(q_heads + 2 heads) * dim] of the tokens at positions pos [n] of sequences seq [n]:
        queries and keys normed (q_norm, k_norm [dim] float32, or None) and rotated (the first rot
        values, all of them by default; pairs "halves" or "adjacent"); queries into q [n][q_heads][dim], keys and values
        into the cache, keys into k [n][heads][dim] too if given (ocr_kv_append_device)."""
        ctx, types = self.ctx, _F16
        rot = self.dim if rot is None else rot
        if pairs in _PAIRS and _native("append", ctx, self._at, table, seq, pos, qkv, q, k, q_norm, k_norm, eps, rot, theta, _PAIRS[pairs]):
            return
        qp, n, q_heads, dim, stride = _tokens(ctx, q, "queries", types, dim=self.dim)
        if stride != q_heads * dim:
            raise _error("queries: its values do not lie one after another")
        width = (q_heads + 2 * self.heads) * dim
        _device(ctx, qkv, "projections")
        code = _code(qkv, "projections")
        if code not in _ANY or tuple(qkv.shape) != (n, width) or (n and qkv.stride()[1] != 1):
            raise _error(f"projections: rows [{n}][{width}] of f32, f16 or bf16 are wanted, not {tuple(qkv.shape)} of {qkv.dtype}")
        if pairs not in _PAIRS:
            raise _error(f'pairs: "halves" or "adjacent" is wanted, not {pairs!r}')
        if theta <= 0 or not 0 <= rot < 2 ** 32:
            raise _error(f"a rotation of {rot} values to the base {theta}")
        out = _code(q, "queries")
        args = ocr_kv_append_args(_array(ctx, seq, "sequence numbers", _I32, (n,)), _array(ctx, pos, "positions", _I32, (n,)),
                                  qkv.data_ptr() or None, code, n, q_heads, qkv.stride()[0] if n > 1 else width,
                                  _array(ctx, q_norm, "q_norm", _F32, (dim,)), _array(ctx, k_norm, "k_norm", _F32, (dim,)), eps, rot,
                                  theta, _PAIRS[pairs], qp, _array(ctx, k, "keys", (out,), (n, self.heads, dim)), out)
        _call("ocr_kv_append_device", ctx.handle, ctypes.byref(self._c), ctypes.byref(self._table(table)), ctypes.byref(args))

    def read(self, table, lens, k, v):
        """The cached keys and values of every sequence's first positions into k and v
        [sequences][positions][heads][dim] (float16 or bfloat16), zeros past its length (lens
        [sequences]; ocr_kv_read_device)."""
        if _native("read", self.ctx, self._at, table, lens, k, v):
            return
        t = self._table(table)
        if len(k.shape) != 4:
            raise _error(f"keys: shape [sequences][positions][heads][dim] is wanted, not {tuple(k.shape)}")
        shape = (t.rows, k.shape[1], self.heads, self.dim)
        kp = _array(self.ctx, k, "keys", _F16, shape)
        code = _code(k, "keys")
        _call("ocr_kv_read_device", self.ctx.handle, ctypes.byref(self._c), ctypes.byref(t),
              _array(self.ctx, lens, "lengths", _I32, (t.rows,)), shape[1], code, kp, _array(self.ctx, v, "values", (code,), shape))

    def attend(self, table, lens, q, out, scale: float | None = None, cap: float = 0.0, slopes=None):
        """Attention of every sequence's last token (lens [sequences] counts it) over its cached
        vectors: q, out [sequences][q_heads][dim] (ocr_decode_attention_device)."""
        ctx = self.ctx
        scale = self.dim ** -0.5 if scale is None else scale
        if _native("attend", ctx, self._at, table, lens, q, out, scale, cap, slopes):
            return
        t = self._table(table)
        qp, n, q_heads, dim, qs = _tokens(ctx, q, "queries", _F16, n=t.rows, dim=self.dim)
        code = _code(q, "queries")
        op, _, _, _, os = _tokens(ctx, out, "outputs", (code,), n, q_heads, dim)
        args = ocr_decode_args(_array(ctx, lens, "lengths", _I32, (n,)), qp, op, code, q_heads, qs, os,
                               scale, cap, _array(ctx, slopes, "slopes", _F32, (q_heads,)))
        _call("ocr_decode_attention_device", ctx.handle, ctypes.byref(self._c), ctypes.byref(t), ctypes.byref(args))

    def fork(self, table, lens, parents, spare, table_out, lens_out, used):
        """The tables and lengths of every group's beams after a step that continued `parents`
        [groups][beams]: whole pages shared, part-filled ones copied into spare [sequences] for all
        but their first child; used [sequences] says where that was (ocr_kv_fork_device)."""
        if _native("fork", self.ctx, self._at, table, lens, parents, spare, table_out, lens_out, used):
            return
        ctx, t = self.ctx, self._table(table)
        if len(parents.shape) != 2 or parents.shape[0] * parents.shape[1] != t.rows:
            raise _error(f"parents: shape [groups][beams] of {t.rows} sequences is wanted, not {tuple(parents.shape)}")
        one = lambda x, what: _array(ctx, x, what, _I32, (t.rows,))  # noqa: E731
        _call("ocr_kv_fork_device", ctx.handle, ctypes.byref(self._c), ctypes.byref(t), one(lens, "lengths"),
              _array(ctx, parents, "parents", _I32, tuple(parents.shape)), parents.shape[1], one(spare, "spare pages"),
              _array(ctx, table_out, "the new table", _I32, (t.rows, t.width)), one(lens_out, "the new lengths"), one(used, "used"))


def attention(ctx, q, k, v, out, docs=None, prefix=None, scale: float | None = None, cap: float = 0.0, slopes=None):
    """Attention over packed documents (ocr_attention_device): q, out [n][q_heads][dim], k, v
    [n][kv_heads][dim], docs [documents + 1] rising offsets (None: one document), prefix
    [documents] tokens at each one's start that all of it sees, slopes [q_heads] of the distance
    bias, cap of the scores' tanh (0: none)."""
    if scale is None:
        scale = q.shape[2] ** -0.5 if len(q.shape) == 3 and q.shape[2] else 1.0
    if _native("attention", ctx, q, k, v, out, docs, prefix, scale, cap, slopes):
        return
    qp, n, q_heads, dim, qs = _tokens(ctx, q, "queries", _F16)
    code = _code(q, "queries")
    kp, _, kv_heads, _, ks = _tokens(ctx, k, "keys", (code,), n, dim=dim)
    vp, _, _, _, vs = _tokens(ctx, v, "values", (code,), n, kv_heads, dim)
    op, _, _, _, os = _tokens(ctx, out, "outputs", (code,), n, q_heads, dim)
    ndocs = 1
    if docs is not None:
        if len(docs.shape) != 1 or docs.shape[0] < 1:
            raise _error(f"documents: offsets [documents + 1] are wanted, not {tuple(docs.shape)}")
        ndocs = docs.shape[0] - 1
    args = ocr_attention_args(qp, kp, vp, op, code, n, q_heads, kv_heads, dim, qs, ks, vs, os,
                              None if docs is None else _array(ctx, docs, "documents", _I32, (ndocs + 1,)), ndocs,
                              _array(ctx, prefix, "prefix", _I32, (ndocs,)), scale, cap,
                              _array(ctx, slopes, "slopes", _F32, (q_heads,)))
    _call("ocr_attention_device", ctx.handle, ctypes.byref(args))


def beam_select(ctx, logits, scores, finished, eos: int | None, out_scores, parents, tokens, out_finished=None):
    """A step of beam search (ocr_beam_select_device): logits [groups * beams][vocab], scores
    [groups][beams] float32, finished [groups][beams] int32 or None, the end token or None; the
    best continuations of every group into out_scores, parents, tokens and out_finished
    [groups][beams]."""
    if _native("beam_select", ctx, logits, scores, finished, eos, out_scores, parents, tokens, out_finished):
        return
    if len(scores.shape) != 2 or len(logits.shape) != 2:
        raise _error(f"logits [groups * beams][vocab] and scores [groups][beams] are wanted, not {tuple(logits.shape)} and {tuple(scores.shape)}")
    shape = tuple(scores.shape)
    rows, vocab = logits.shape
    _device(ctx, logits, "logits")
    code = _code(logits, "logits")
    if code not in _ANY or rows != shape[0] * shape[1] or (rows and vocab > 1 and logits.stride()[1] != 1):
        raise _error(f"logits: {shape[0] * shape[1]} rows of f32, f16 or bf16 are wanted, not {tuple(logits.shape)} of {logits.dtype}")
    if eos is not None and not -2 ** 31 <= eos < 2 ** 31:
        raise _error(f"the end token {eos} is not in the vocabulary")
    arr = lambda x, what, types: _array(ctx, x, what, types, shape)  # noqa: E731
    args = ocr_beam_args(logits.data_ptr() or None, code, shape[0], shape[1], vocab, logits.stride()[0] if rows > 1 else vocab,
                         arr(scores, "scores", _F32), arr(finished, "finished", _I32), -1 if eos is None else eos,
                         arr(out_scores, "new scores", _F32), arr(parents, "parents", _I32), arr(tokens, "tokens", _I32),
                         arr(out_finished, "new finished", _I32))
    _call("ocr_beam_select_device", ctx.handle, ctypes.byref(args))
