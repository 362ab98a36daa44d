"""A text decoder's operators (include/ocrhip.h): a paged cache of keys and values, attention over
prompts and of single tokens over the cache, beam search; rotary positions of several axes, eviction
from the cache by the attention weight that its keys got, latent attention.

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


class ocr_axes(ctypes.Structure):
    _fields_ = [("at", P), ("count", U32), ("pairs", U32 * 4), ("in_turn", I32), ("own_ladder", I32)]


class ocr_rotate_args(ctypes.Structure):
    _fields_ = [("x", P), ("out", P), ("type", I32), ("n", U32), ("heads", U32), ("dim", U32), ("x_stride", I64), ("x_head", I64),
                ("out_stride", I64), ("out_head", I64), ("first", U32), ("rot", U32), ("theta", F64), ("adjacent", I32), ("back", I32)]


class ocr_evict_args(ctypes.Structure):
    _fields_ = [("lens", P), ("newest", P), ("weights", P), ("held", P), ("most", U32), ("keep", U32), ("first", U32), ("recent", U32),
                ("weights_out", P), ("held_out", P), ("lens_out", P)]


class ocr_latent_cache(ctypes.Structure):
    _fields_ = [("data", P), ("pages", U32), ("page", U32), ("rank", U32), ("rot", U32), ("type", I32)]


class ocr_latent_append_args(ctypes.Structure):
    _fields_ = [("seq", P), ("pos", P), ("x", P), ("type", I32), ("n", U32), ("stride", I64), ("norm", P), ("eps", F32), ("theta", F64),
                ("adjacent", I32), ("out", P)]


class ocr_latent_decode_args(ctypes.Structure):
    _fields_ = [("lens", P), ("q", P), ("out", P), ("heads", U32), ("q_stride", I64), ("out_stride", I64), ("scale", F32)]


class ocr_latent_attention_args(ctypes.Structure):
    _fields_ = [("q", P), ("k", P), ("r", P), ("v", P), ("out", P), ("type", I32), ("n", U32), ("heads", U32), ("key", U32), ("rot", U32),
                ("value", U32), ("q_stride", I64), ("k_stride", I64), ("k_head", I64), ("r_stride", I64), ("v_stride", I64),
                ("v_head", I64), ("out_stride", I64), ("docs", P), ("ndocs", U32), ("prefix", P), ("scale", F32)]


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
                      for f in ("kv_append", "kv_read", "attention", "decode_attention", "beam_select", "kv_fork", "kv_append_axes", "rotate",
                                "attention_weights", "decode_attention_weights", "kv_evict", "latent_append", "latent_decode",
                                "latent_attention")])
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


def _heads(ctx, x, what, types, n=None, heads=None, dim=None):
    """(address, tokens, heads, dim, stride, head stride) of x [tokens][heads][dim], whose tokens and heads may lie apart."""
    _device(ctx, x, what)
    if _code(x, what) not in types:
        raise _error(f"{what}: {' or '.join(_NAMES[t] for t in types)} is wanted, not {x.dtype}")
    shape, strides = x.shape, x.stride()
    if len(shape) != 3 or any(w is not None and w != v for w, v in zip((n, heads, dim), shape)):
        want = tuple("any" if v is None else v for v in (n, heads, dim))
        raise _error(f"{what}: shape {want} is wanted, not {tuple(shape)}")
    n, heads, dim = shape
    if n and dim > 1 and strides[2] != 1:
        raise _error(f"{what}: a head's values do not lie one after another")
    head = strides[1] if heads > 1 else dim
    return x.data_ptr() or None, n, heads, dim, strides[0] if n > 1 else max((heads - 1) * head + dim, 0), head


_I32, _F32, _F16, _ANY = (5,), (0,), (1, 2), (0, 1, 2)
_PAIRS = {"halves": False, "adjacent": True}
_ORDERS, _LADDERS = {"blocks": False, "turns": True}, {"shared": False, "own": True}


def _places(x, what):
    if len(x.shape) != 3:
        raise _error(f"{what}: three dimensions are wanted, not {tuple(x.shape)}")
    return tuple(x.shape)


def _pairs_of(axes, count, rot):
    """How many pairs of a rotation each axis has: the caller's, or as many each."""
    if axes is None:
        if count < 1 or rot // 2 % count:
            raise _error(f"axes: a rotation of {rot} values in {count} equal parts")
        return (rot // 2 // count,) * count
    axes = tuple(axes)
    if not 1 <= len(axes) <= 4 or any(not 0 <= v < 2 ** 32 for v in axes):
        raise _error(f"axes: 1 to 4 numbers of pairs are wanted, not {axes}")
    if count != len(axes):
        raise _error(f"positions of {count} axes, and pairs of {len(axes)}")
    return axes


def _axes(ctx, at, axes, order, ladder, rot, n):
    """The C ABI's axes of positions at [n][axes], or [n] for one."""
    if order not in _ORDERS or ladder not in _LADDERS:
        raise _error(f'axes in "blocks" or in "turns", a "shared" or an "own" ladder are wanted, not {order!r} and {ladder!r}')
    if len(at.shape) not in (1, 2):
        raise _error(f"positions: shape [{n}][axes] is wanted, not {tuple(at.shape)}")
    count = at.shape[1] if len(at.shape) == 2 else 1
    pairs = _pairs_of(axes, count, rot)
    shape = (n, count) if len(at.shape) == 2 else (n,)
    return ocr_axes(_array(ctx, at, "positions", _I32, shape), count, (U32 * 4)(*pairs), _ORDERS[order], _LADDERS[ladder])


def _turn(pairs, theta, rot):
    if pairs not in _PAIRS:
        raise _error(f'pairs: "halves" or "adjacent" is wanted, not {pairs!r}')
    if theta <= 0 or not 0 <= rot < 2 ** 32:
        raise _error(f"a rotation of {rot} values to the base {theta}")
    return _PAIRS[pairs]


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
               theta: float = 1e4, pairs: str = "halves", at=None, axes=None, order: str = "blocks", ladder: str = "shared"):
        """Projections qkv [n][(q_heads + 2 heads) * dim] of the tokens at positions pos [n] of sequences seq [n]:
        queries and keys normed (q_norm, k_norm [dim] float32, or None) and rotated (the first rot
        values, all of them by default; pairs "halves" or "adjacent"); queries into q [n][q_heads][dim], keys and values
        into the cache, keys into k [n][heads][dim] too if given (ocr_kv_append_device). With at [n][axes]
        (int32) the rotation goes by those positions instead, as rotate() does with axes, order and ladder
        (ocr_kv_append_axes_device)."""
        ctx, types = self.ctx, _F16
        rot = self.dim if rot is None else rot
        if at is not None:
            if pairs in _PAIRS and order in _ORDERS and ladder in _LADDERS and _native(
                    "append_axes", ctx, self._at, table, seq, pos, qkv, q, k, q_norm, k_norm, eps, rot, theta, _PAIRS[pairs], at, axes,
                    _ORDERS[order], _LADDERS[ladder]):
                return
        elif axes is not None:
            raise _error("axes without positions (at)")
        elif pairs in _PAIRS and _native("append", ctx, self._at, table, seq, pos, qkv, q, k, q_norm, k_norm, eps, rot, theta, _PAIRS[pairs]):
            return
        qp, n, q_heads, dim, stride = _tokens(ctx, q, "queries", types, dim=self.dim)
        if stride != q_heads * dim:
            raise _error("queries: its values do not lie one after another")
        width = (q_heads + 2 * self.heads) * dim
        _device(ctx, qkv, "projections")
        code = _code(qkv, "projections")
        if code not in _ANY or tuple(qkv.shape) != (n, width) or (n and qkv.stride()[1] != 1):
            raise _error(f"projections: rows [{n}][{width}] of f32, f16 or bf16 are wanted, not {tuple(qkv.shape)} of {qkv.dtype}")
        adjacent = _turn(pairs, theta, rot)
        out = _code(q, "queries")
        args = ocr_kv_append_args(_array(ctx, seq, "sequence numbers", _I32, (n,)), _array(ctx, pos, "positions", _I32, (n,)),
                                  qkv.data_ptr() or None, code, n, q_heads, qkv.stride()[0] if n > 1 else width,
                                  _array(ctx, q_norm, "q_norm", _F32, (dim,)), _array(ctx, k_norm, "k_norm", _F32, (dim,)), eps, rot,
                                  theta, adjacent, qp, _array(ctx, k, "keys", (out,), (n, self.heads, dim)), out)
        where = ctypes.byref(self._c), ctypes.byref(self._table(table)), ctypes.byref(args)
        if at is None:
            _call("ocr_kv_append_device", ctx.handle, *where)
        else:
            _call("ocr_kv_append_axes_device", ctx.handle, *where, ctypes.byref(_axes(ctx, at, axes, order, ladder, rot, n)))

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

    def attend(self, table, lens, q, out, scale: float | None = None, cap: float = 0.0, slopes=None, weights=None):
        """Attention of every sequence's last token (lens [sequences] counts it) over its cached
        vectors: q, out [sequences][q_heads][dim] (ocr_decode_attention_device). What each key got is
        added to weights [sequences][heads][places] float32 if given, its query heads together
        (ocr_decode_attention_weights_device)."""
        ctx = self.ctx
        scale = self.dim ** -0.5 if scale is None else scale
        if _native("attend", ctx, self._at, table, lens, q, out, scale, cap, slopes, weights):
            return
        t = self._table(table)
        qp, n, q_heads, dim, qs = _tokens(ctx, q, "queries", _F16, n=t.rows, dim=self.dim)
        code = _code(q, "queries")
        op, _, _, _, os = _tokens(ctx, out, "outputs", (code,), n, q_heads, dim)
        args = ocr_decode_args(_array(ctx, lens, "lengths", _I32, (n,)), qp, op, code, q_heads, qs, os,
                               scale, cap, _array(ctx, slopes, "slopes", _F32, (q_heads,)))
        if weights is None:
            _call("ocr_decode_attention_device", ctx.handle, ctypes.byref(self._c), ctypes.byref(t), ctypes.byref(args))
            return
        most = _places(weights, "weights")[2]
        _call("ocr_decode_attention_weights_device", ctx.handle, ctypes.byref(self._c), ctypes.byref(t), ctypes.byref(args),
              _array(ctx, weights, "weights", _F32, (n, self.heads, most)), most)

    def evict(self, table, lens, newest, weights, held, keep: int, lens_out, first: int = 0, recent: int = 0, weights_out=None,
              held_out=None):
        """Drops cached tokens until `keep` of a sequence's (lens [sequences]) are left, each head its own: the
        least of weights [sequences][heads][places] (float32, what attend() and attention() add up), but none at a position
        under `first` and none of the `recent` last up to newest [sequences], the position of its newest token. held, as
        weights but int32, says which position the token at a place has, or less than 0 as long as no
        eviction has said so. New lengths into lens_out, weights and positions into weights_out and held_out, by default
        over the old ones; the kept vectors are in places 0 to the new length (ocr_kv_evict_device)."""
        ctx = self.ctx
        weights_out, held_out = weights if weights_out is None else weights_out, held if held_out is None else held_out
        if _native("evict", ctx, self._at, table, lens, newest, weights, held, keep, lens_out, first, recent, weights_out, held_out):
            return
        t = self._table(table)
        most = _places(weights, "weights")[2]
        if any(not 0 <= v < 2 ** 32 for v in (keep, first, recent)):
            raise _error(f"eviction: {keep} tokens to keep, {first} first and {recent} recent ones")
        row = lambda x, what: _array(ctx, x, what, _I32, (t.rows,))  # noqa: E731
        cell = lambda x, what, types: _array(ctx, x, what, types, (t.rows, self.heads, most))  # noqa: E731
        args = ocr_evict_args(row(lens, "lengths"), row(newest, "newest positions"), cell(weights, "weights", _F32), cell(held, "positions", _I32),
                              most, keep, first, recent, cell(weights_out, "new weights", _F32), cell(held_out, "new positions", _I32),
                              row(lens_out, "the new lengths"))
        _call("ocr_kv_evict_device", ctx.handle, ctypes.byref(self._c), ctypes.byref(t), ctypes.byref(args))

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


class LatentCache:
    """A paged cache of latent vectors: pages of `page` positions that hold rank + rot values a token of type "f16" or
    "bf16" (ocr_latent_cache). memory: the caller's [pages][page][rank + rot]; without it the cache allocates its
    own. Tables as a KvCache's."""

    _table = KvCache._table

    def __init__(self, ctx, pages: int, page: int, rank: int, rot: int, dtype: str = "bf16", memory=None):
        if dtype not in ("f16", "bf16"):
            raise _error(f"latent cache: f16 or bf16 is wanted, not {dtype!r}")
        if min(pages, page, rank) < 1 or rot < 0:
            raise _error("latent cache: empty")
        if max(pages, page, rank, rot) >= 2 ** 32:
            raise _error(f"latent cache: sizes {(pages, page, rank, rot)} are past 32 bits")
        self.ctx, self.pages, self.page, self.rank, self.rot, self.dtype = ctx, pages, page, rank, rot, dtype
        shape, code = (pages, page, rank + rot), _SHORT[dtype]
        self.data = DeviceArray(ctx.alloc(pages * page * (rank + rot) * 2), shape, dtype) if memory is None else memory
        self._c = ocr_latent_cache(_array(ctx, self.data, "latent cache", (code,), shape), pages, page, rank, rot, code)
        self._at = ctypes.addressof(self._c)

    def append(self, table, seq, pos, x, out=None, norm=None, eps: float = 1e-6, theta: float = 1e4, pairs: str = "halves", at=None,
               axes=None, order: str = "blocks", ladder: str = "shared"):
        """Projections x [n][rank + rot] of the tokens at positions pos [n] of sequences seq [n]: the first rank values normed
        (norm [rank] float32, or None), the others rotated by pos, or by at [n][axes] as rotate() does; into the
        cache, and into out [n][rank + rot] of its type if given (ocr_latent_append_device)."""
        ctx = self.ctx
        if at is None and axes is not None:
            raise _error("axes without positions (at)")
        if pairs in _PAIRS and order in _ORDERS and ladder in _LADDERS and _native(
                "latent_append", ctx, self._at, table, seq, pos, x, out, norm, eps, theta, _PAIRS[pairs], at, axes, _ORDERS[order],
                _LADDERS[ladder]):
            return
        width = self.rank + self.rot
        _device(ctx, x, "projections")
        code = _code(x, "projections")
        if code not in _ANY or len(x.shape) != 2 or x.shape[1] != width or (x.shape[0] and width > 1 and x.stride()[1] != 1):
            raise _error(f"projections: rows [tokens][{width}] of f32, f16 or bf16 are wanted, not {tuple(x.shape)} of {x.dtype}")
        n = x.shape[0]
        adjacent = _turn(pairs, theta, self.rot)
        args = ocr_latent_append_args(_array(ctx, seq, "sequence numbers", _I32, (n,)), _array(ctx, pos, "positions", _I32, (n,)),
                                      x.data_ptr() or None, code, n, x.stride()[0] if n > 1 else width,
                                      _array(ctx, norm, "norm", _F32, (self.rank,)), eps, theta, adjacent,
                                      _array(ctx, out, "outputs", (self._c.type,), (n, width)))
        turn = None if at is None else ctypes.byref(_axes(ctx, at, axes, order, ladder, self.rot, n))
        _call("ocr_latent_append_device", ctx.handle, ctypes.byref(self._c), ctypes.byref(self._table(table)), ctypes.byref(args), turn)

    def attend(self, table, lens, q, out, scale: float):
        """Attention of every sequence's last token (lens [sequences] counts it) over its latent vectors: q
        [sequences][heads][rank + rot] with the keys' expansion absorbed, out [sequences][heads][rank], the values' expansion to
        follow (ocr_latent_decode_device)."""
        ctx = self.ctx
        if _native("latent_attend", ctx, self._at, table, lens, q, out, scale):
            return
        t, code = self._table(table), self._c.type
        qp, n, heads, _, qs = _tokens(ctx, q, "queries", (code,), n=t.rows, dim=self.rank + self.rot)
        op, _, _, _, os = _tokens(ctx, out, "outputs", (code,), n, heads, self.rank)
        args = ocr_latent_decode_args(_array(ctx, lens, "lengths", _I32, (n,)), qp, op, heads, qs, os, scale)
        _call("ocr_latent_decode_device", ctx.handle, ctypes.byref(self._c), ctypes.byref(t), ctypes.byref(args))

    def fork(self, table, lens, parents, spare, table_out, lens_out, used):
        """As KvCache.fork (ocr_latent_fork_device)."""
        ctx, t = self.ctx, self._table(table)
        if len(parents.shape) != 2 or parents.shape[0] * parents.shape[1] != t.rows:
            raise _error(f"parents: shape [groups][beams] of {t.rows} sequences is wanted, not {tuple(parents.shape)}")
        one = lambda x, what: _array(ctx, x, what, _I32, (t.rows,))  # noqa: E731
        _call("ocr_latent_fork_device", ctx.handle, ctypes.byref(self._c), ctypes.byref(t), one(lens, "lengths"),
              _array(ctx, parents, "parents", _I32, tuple(parents.shape)), parents.shape[1], one(spare, "spare pages"),
              _array(ctx, table_out, "the new table", _I32, (t.rows, t.width)), one(lens_out, "the new lengths"), one(used, "used"))


def rotate(ctx, x, at, out=None, first: int = 0, rot: int | None = None, theta: float = 1e4, pairs: str = "halves", axes=None,
           order: str = "blocks", ladder: str = "shared", back: bool = False):
    """Rotary positions of one or several axes (ocr_rotate_device): x [n][heads][dim] with its values from `first` on, rot of them (all by
    default), rotated by positions at [n][axes] (int32; [n] for one axis) into out, or in place. axes: how many pairs each
    axis has (as many each by default), in "blocks" or one after another in "turns"; the frequencies fall over all pairs
    ("shared") or over each axis' own ("own"). back: the other way, which is also the gradient."""
    out = x if out is None else out
    rot = (x.shape[2] if len(x.shape) == 3 else 0) - first if rot is None else rot
    if pairs in _PAIRS and order in _ORDERS and ladder in _LADDERS and _native("rotate", ctx, x, at, out, first, rot, theta, _PAIRS[pairs],
                                                                               axes, _ORDERS[order], _LADDERS[ladder], bool(back)):
        return
    xp, n, heads, dim, xs, xh = _heads(ctx, x, "inputs", _ANY)
    code = _code(x, "inputs")
    op, _, _, _, os, oh = _heads(ctx, out, "outputs", (code,), n, heads, dim)
    adjacent = _turn(pairs, theta, rot)
    if not 0 <= first < 2 ** 32:
        raise _error(f"a rotation from value {first} on")
    args = ocr_rotate_args(xp, op, code, n, heads, dim, xs, xh, os, oh, first, rot, theta, adjacent, bool(back))
    _call("ocr_rotate_device", ctx.handle, ctypes.byref(args), ctypes.byref(_axes(ctx, at, axes, order, ladder, rot, n)))


def _documents(ctx, docs, prefix):
    """The C ABI's documents: offsets, how many, prefixes."""
    ndocs = 1
    if docs is not None:
        if len(docs.shape) != 1 or docs.shape[0] < 1:
            raise _error(f"documents: offsets [documents + 1] are wanted, not {tuple(docs.shape)}")
        ndocs = docs.shape[0] - 1
    return None if docs is None else _array(ctx, docs, "documents", _I32, (ndocs + 1,)), ndocs, _array(ctx, prefix, "prefix", _I32, (ndocs,))


def latent_attention(ctx, q, k, r, v, out, docs=None, prefix=None, scale: float | None = None):
    """Latent attention over packed documents with expanded keys and values (ocr_latent_attention_device): q
    [n][heads][key + rot], k [n][heads][key] and r [n][rot] that all heads share (None: no such part), v, out [n][heads][value];
    k and v may lie beside each other, r beside the latent vectors. Documents as in attention()."""
    if scale is None:
        scale = q.shape[2] ** -0.5 if len(q.shape) == 3 and q.shape[2] else 1.0
    if _native("latent_attention", ctx, q, k, r, v, out, docs, prefix, scale):
        return
    qp, n, heads, width, qs = _tokens(ctx, q, "queries", _F16)
    code = _code(q, "queries")
    kp, _, _, key, ks, kh = _heads(ctx, k, "keys", (code,), n, heads)
    vp, _, _, value, vs, vh = _heads(ctx, v, "values", (code,), n, heads)
    op, _, _, _, os = _tokens(ctx, out, "outputs", (code,), n, heads, value)
    rp, rot, rs = None, width - key, 0
    if r is not None:
        _device(ctx, r, "shared keys")
        if _code(r, "shared keys") != code or tuple(r.shape) != (n, rot) or (n and rot > 1 and r.stride()[1] != 1):
            raise _error(f"shared keys: rows [{n}][{rot}] of {_NAMES[code]} are wanted, not {tuple(r.shape)} of {r.dtype}")
        rp, rs = r.data_ptr() or None, r.stride()[0] if n > 1 else rot
    elif rot:
        raise _error(f"queries of {width} values over keys of {key}, and no shared keys")
    args = ocr_latent_attention_args(qp, kp, rp, vp, op, code, n, heads, key, rot, value, qs, ks, kh, rs, vs, vh, os,
                                     *_documents(ctx, docs, prefix), scale)
    _call("ocr_latent_attention_device", ctx.handle, ctypes.byref(args))


def attention(ctx, q, k, v, out, docs=None, prefix=None, scale: float | None = None, cap: float = 0.0, slopes=None, weights=None,
              window: int | None = None):
    """Attention over packed documents (ocr_attention_device): q, out [n][q_heads][dim], k, v
    [n][kv_heads][dim], docs [documents + 1] rising offsets (None: one document), prefix
    [documents] tokens at each one's start that all of it sees, slopes [q_heads] of the distance
    bias, cap of the scores' tanh (0: none). What each key got from its document's queries (the last `window` of
    them; None: all) is added to weights [documents][kv_heads][places] float32 if given (ocr_attention_weights_device)."""
    if scale is None:
        scale = q.shape[2] ** -0.5 if len(q.shape) == 3 and q.shape[2] else 1.0
    if window is not None and (weights is None or not 1 <= window < 2 ** 31):
        raise _error(f"a window of {window} queries without weights" if weights is None else f"a window of {window} queries")
    if _native("attention", ctx, q, k, v, out, docs, prefix, scale, cap, slopes, weights, 0 if window is None else window):
        return
    qp, n, q_heads, dim, qs = _tokens(ctx, q, "queries", _F16)
    code = _code(q, "queries")
    kp, _, kv_heads, _, ks = _tokens(ctx, k, "keys", (code,), n, dim=dim)
    vp, _, _, _, vs = _tokens(ctx, v, "values", (code,), n, kv_heads, dim)
    op, _, _, _, os = _tokens(ctx, out, "outputs", (code,), n, q_heads, dim)
    documents = _documents(ctx, docs, prefix)
    args = ocr_attention_args(qp, kp, vp, op, code, n, q_heads, kv_heads, dim, qs, ks, vs, os, *documents, scale, cap,
                              _array(ctx, slopes, "slopes", _F32, (q_heads,)))
    if weights is None:
        _call("ocr_attention_device", ctx.handle, ctypes.byref(args))
        return
    most = _places(weights, "weights")[2]
    _call("ocr_attention_weights_device", ctx.handle, ctypes.byref(args),
          _array(ctx, weights, "weights", _F32, (documents[1], kv_heads, most)), most, window or 0)


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
