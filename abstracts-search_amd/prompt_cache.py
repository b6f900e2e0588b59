"""The keys and values of prompts in pages, and the attention of texts that stand behind one of them.

A causal encoder computes the same hidden states for a prompt whatever text follows it, so texts behind one prompt need the
prompt's keys and values once.  ``PromptCache`` holds them (C ABI: ``include/mi_encoder.h``, kernels:
``csrc/prompt_kernels.h``)::

    cache = PromptCache(n_layers=28, n_kv_heads=2, head_dim=128, n_pages=256)
    prompt = cache.new()
    cache.extend(prompt, k, v)                        # [n_layers, n, n_kv_heads, head_dim]
    out = cache.attention(prompt, layer, q, k, v, cu_q, cu_k)
    variants = cache.fork(prompt, 4)                  # full pages shared, the last page's tokens copied
    cache.free(prompt)

``SentenceTransformer.cache_prompt`` keeps one of these for a causal model and encodes prompted texts through it.  There is
no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math
import struct
import weakref
from ctypes import POINTER, c_int, c_int32, c_int64, c_void_p

from . import _native

PAGE = 64                                            # tokens of a page (MI_PROMPT_PAGE)


class _Cfg(ctypes.Structure):
    _fields_ = [(n, c_int32) for n in ("n_layers", "n_kv_heads", "head_dim", "dtype", "n_pages", "max_entries", "max_tokens")]


_Strides = c_int64 * 3
# mi_prompt_attn, field by field
_ATTN = struct.Struct("@6i4P8q2PifiiPq")


class _Lib:
    _lib = None

    @classmethod
    def get(cls):
        if cls._lib is None:
            lib = _native.load("encoder")
            lib.mi_enc_last_error.restype = ctypes.c_char_p
            v, i32, pi32 = c_void_p, c_int32, POINTER(c_int32)
            sigs = {
                "mi_prompt_cache_create": [POINTER(_Cfg), c_int, v, POINTER(v)],
                "mi_prompt_cache_destroy": [v],
                "mi_prompt_cache_new": [v, v, pi32],
                "mi_prompt_cache_reserve": [v, i32, i32, v],
                "mi_prompt_cache_write": [v, i32, i32, i32, i32, i32, v, POINTER(c_int64), v, POINTER(c_int64), v],
                "mi_prompt_cache_extend": [v, i32, i32, v, POINTER(c_int64), v, POINTER(c_int64), v],
                "mi_prompt_cache_fork": [v, i32, i32, pi32, pi32, v],
                "mi_prompt_cache_copy": [v, i32, pi32, v],
                "mi_prompt_cache_free": [v, i32, pi32, v],
                "mi_prompt_cache_compact": [v, v, pi32],
                "mi_prompt_cache_resize": [v, v, i32, v],
                "mi_prompt_cache_entry": [v, i32, pi32, pi32, i32],
                "mi_prompt_cache_used": [v, pi32, pi32],
                "mi_prompt_attention_workspace": [v, v, POINTER(c_int64)],
                "mi_prompt_attention": [v, v, v],
            }
            for name, args in sigs.items():
                fn = getattr(lib, name)
                fn.argtypes = args
                fn.restype = c_int
            cls._lib = lib
        return cls._lib


def _check(rc: int):
    if rc != 0:
        raise RuntimeError("mi_prompt_cache: " + _Lib.get().mi_enc_last_error().decode())


def _int32(what, *numbers):
    """refuses what ctypes would cut to 32 bits (n >> 31 is 0 for the ordinary ones: the short way past it)"""
    for n in numbers:
        if not -1 << 31 <= n < 1 << 31:
            raise ValueError(f"PromptCache.{what}: {n} is no int32")


def _no_gradient(what, *tensors):
    """refuses tensors whose gradient (of either mode) would be lost"""
    import torch
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"PromptCache.{what} has no gradient: call it under torch.no_grad()")
    forward = torch.autograd.forward_ad
    if getattr(forward, "_current_level", 0) >= 0 and any(t is not None and forward.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"PromptCache.{what} has no gradient: a tensor carries a forward-mode tangent")


def _destroy(handle):
    try:
        _Lib.get().mi_prompt_cache_destroy(handle)
    except Exception:
        pass


class PromptCache:
    """A pool of ``n_pages`` pages of 64 tokens: ``pages`` [n_pages, n_layers, n_kv_heads, 2 (K, V), 64, head_dim].

    ``dtype``: torch.bfloat16 or torch.float16; ``max_entries``: prompts held at a time; ``max_tokens``: of one prompt (None:
    whatever the pages hold at first).  Every call works on torch's current stream of the cache's device.  An entry belongs to the
    stream it was made on; other streams may read it once the caller has ordered them behind its writes."""

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, n_pages: int, dtype=None, device=None,
                 max_entries: int = 256, max_tokens: int | None = None):
        import torch
        dtype = torch.bfloat16 if dtype is None else dtype
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"PromptCache: dtype must be torch.bfloat16 or torch.float16, got {dtype}")
        if head_dim not in (64, 128):
            raise ValueError(f"PromptCache: head_dim must be 64 or 128, got {head_dim}")
        for name, n in (("n_layers", n_layers), ("n_kv_heads", n_kv_heads), ("n_pages", n_pages), ("max_entries", max_entries)):
            if not 1 <= n < 1 << 31:
                raise ValueError(f"PromptCache: {name} must be positive (and an int32), got {n}")
        if max_tokens is not None and not 1 <= max_tokens < 1 << 31:
            raise ValueError(f"PromptCache: max_tokens must be positive (and an int32), got {max_tokens}")
        lib = _Lib.get()
        if not torch.cuda.is_available():
            raise RuntimeError("mi_prompt_cache: no HIP device available: the MI355X prompt cache has no CPU fallback")
        dev = torch.device("cuda" if device is None else device if not isinstance(device, int) else f"cuda:{device}")
        if dev.type != "cuda":
            raise ValueError(f"PromptCache: a GPU device, got {dev}")
        self.device = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
        self.dtype, self.n_layers, self.n_kv_heads, self.head_dim = dtype, n_layers, n_kv_heads, head_dim
        self.pages = torch.zeros((n_pages, n_layers, n_kv_heads, 2, PAGE, head_dim), dtype=dtype, device=self.device)
        cfg = _Cfg(n_layers, n_kv_heads, head_dim, 1 if dtype == torch.bfloat16 else 2, n_pages, max_entries, max_tokens or 0)
        self._h = c_void_p()
        _check(lib.mi_prompt_cache_create(ctypes.byref(cfg), self.device.index, self.pages.data_ptr(), ctypes.byref(self._h)))
        self._close = weakref.finalize(self, _destroy, self._h)
        self._lib = lib
        self._max_entries = max_entries
        self._table_cap = -(-max_tokens // PAGE) if max_tokens else n_pages   # pages of the longest entry
        # What is known without asking the library.  Another thread may change it meanwhile: either dict is replaced on both sides of
        # a change, and what was learnt before it goes into the one that was there then.
        self._tables: dict = {}                      # entry -> its table, as far as known: (full pages, the last one or -1), until pages move
        self._plans: dict = {}                       # (entry, shapes) -> bytes of workspace, until an entry's length changes
        # torch's current stream as a pointer (building the Stream object first is 1.7 us of a 10 us call)
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        index, device = self.device.index, self.device
        self._stream = (lambda: raw(index)) if raw else (lambda: torch.cuda.current_stream(device).cuda_stream)

    # -- prompts ------------------------------------------------------------
    def new(self) -> int:
        """an empty entry"""
        e = c_int32()
        _check(self._lib.mi_prompt_cache_new(self._h, self._stream(), ctypes.byref(e)))
        return e.value

    def reserve(self, entry: int, n: int) -> None:
        """n more tokens at the end of the entry, to be filled by ``write``"""
        _int32("reserve", entry, n)
        self._plans = {}
        self._tables.pop(entry, None)
        rc = self._lib.mi_prompt_cache_reserve(self._h, entry, n, self._stream())
        self._plans = {}
        _check(rc)

    def write(self, entry: int, k, v, start: int, layer: int = 0) -> None:
        """keys and values of tokens start .. of layers layer ..: [layers, n, n_kv_heads, head_dim], or one layer without the
        first axis.  Tokens in pages that other entries share are refused.  No gradient."""
        _int32("write", entry, start, layer)
        k, v = self._kv(k, v, "write")
        ks, vs = _Strides(*k.stride()[:3]), _Strides(*v.stride()[:3])
        _check(self._lib.mi_prompt_cache_write(self._h, entry, layer, k.shape[0], start, k.shape[1], k.data_ptr(), ks, v.data_ptr(), vs,
                                               self._stream()))

    def extend(self, entry: int, k, v) -> None:
        """tokens at the end of the entry: k, v [n_layers, n, n_kv_heads, head_dim].  No gradient."""
        if entry >> 31:
            _int32("extend", entry)
        k, v = self._kv(k, v, "extend")
        if k.shape[0] != self.n_layers:
            raise ValueError(f"PromptCache.extend: keys and values of all {self.n_layers} layers, got {tuple(k.shape)}")
        ks, vs = _Strides(*k.stride()[:3]), _Strides(*v.stride()[:3])
        self._plans = {}
        self._tables.pop(entry, None)
        rc = self._lib.mi_prompt_cache_extend(self._h, entry, k.shape[1], k.data_ptr(), ks, v.data_ptr(), vs, self._stream())
        self._plans = {}
        _check(rc)

    def _kv(self, k, v, what):
        import torch
        if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad) or getattr(torch.autograd.forward_ad, "_current_level", 0) >= 0:
            _no_gradient(what, k, v)
        if k.dim() == 3 and v.dim() == 3:
            k, v = k[None], v[None]
        want = (self.n_kv_heads, self.head_dim)
        if k.dim() != 4 or k.shape != v.shape or tuple(k.shape[2:]) != want:
            raise ValueError(f"PromptCache: keys and values [layers, n, {want[0]}, {want[1]}], got {tuple(k.shape)} and {tuple(v.shape)}")
        return self._fit(k, "keys"), self._fit(v, "values")

    def _fit(self, t, what):
        """a tensor the kernels can read: the cache's type and device, 16-byte rows"""
        if t.dtype != self.dtype or t.device != self.device:
            raise ValueError(f"PromptCache: {what} must be {self.dtype} on {self.device}, got {t.dtype} on {t.device}")
        if t.stride(-1) != 1 or t.data_ptr() & 15 or any(s & 7 for s in t.stride()[:-1]):
            t = t.new_empty(t.shape).copy_(t)        # (contiguous() keeps odd strides of axes of length 1, and the address)
        return t

    def fork(self, entry: int, count: int = 1) -> list[int]:
        """`count` new entries that begin as `entry` does: its full pages are shared, the tokens of its last page (and pages that
        a captured `write` reaches) copied"""
        if count < 0:
            raise ValueError(f"PromptCache.fork: count must not be negative, got {count}")
        if entry >> 31:
            _int32("fork", entry)
        if count > self._max_entries:
            raise RuntimeError(f"mi_prompt_cache: prompt cache: more than max_entries ({self._max_entries}) entries")
        out, own, tables = (c_int32 * count)(), (c_int32 * count)(), self._tables
        _check(self._lib.mi_prompt_cache_fork(self._h, entry, count, out, own, self._stream()))
        kids, own = out[:], own[:]
        if count > 1 and own[0] > -2:                # (their tables without asking for each of them)
            full = self.table(kids[0])               # (not the parent's: another thread may extend that)
            if own[0] >= 0:
                full.pop()
            tables.update({k: (full, p) for k, p in zip(kids, own)})
        return kids

    def copy(self, entry: int) -> int:
        """a new entry with the same tokens in pages of its own"""
        if entry >> 31:
            _int32("copy", entry)
        e = c_int32()
        _check(self._lib.mi_prompt_cache_copy(self._h, entry, ctypes.byref(e), self._stream()))
        return e.value

    def free(self, entries) -> None:
        """drops an entry or several; their pages are free once no other entry shares them"""
        entries = [entries] if isinstance(entries, int) else list(entries)
        self._plans = {}
        for e in entries:
            if e >> 31:
                _int32("free", e)
            self._tables.pop(e, None)
        rc = self._lib.mi_prompt_cache_free(self._h, len(entries), (c_int32 * len(entries))(*entries), self._stream())
        self._plans = {}
        _check(rc)

    def compact(self) -> int:
        """moves pages down until the used ones are the first ones of the pool; how many were moved"""
        n = c_int32()
        self._tables = {}
        rc = self._lib.mi_prompt_cache_compact(self._h, self._stream(), ctypes.byref(n))
        self._tables = {}
        _check(rc)
        return n.value

    def resize(self, n_pages: int) -> None:
        """another pool size (at least the used pages): the used pages move to the front of the new pool.  Waits for the
        device; graphs captured over the old pool must not be replayed."""
        import torch
        if not 1 <= n_pages < 1 << 31:
            raise ValueError(f"PromptCache.resize: n_pages must be positive (and an int32), got {n_pages}")
        pages = torch.zeros((n_pages, *self.pages.shape[1:]), dtype=self.dtype, device=self.device)
        self._tables = {}
        rc = self._lib.mi_prompt_cache_resize(self._h, pages.data_ptr(), n_pages, self._stream())
        self._tables = {}
        _check(rc)
        self.pages = pages

    # -- what is held -----------------------------------------------------------
    def length(self, entry: int) -> int:
        _int32("length", entry)
        n = c_int32()
        _check(self._lib.mi_prompt_cache_entry(self._h, entry, ctypes.byref(n), None, 0))
        return n.value

    def table(self, entry: int) -> list[int]:
        """the page numbers of the entry, in order"""
        known = self._tables.get(entry)
        if known is not None:
            full, last = known
            return full + [last] if last >= 0 else full[:]
        if entry >> 31:
            _int32("table", entry)
        cap, n = self._table_cap, c_int32()
        t = (c_int32 * cap)()
        _check(self._lib.mi_prompt_cache_entry(self._h, entry, ctypes.byref(n), t, cap))
        return t[:-(-n.value // PAGE)]

    @property
    def n_pages(self) -> int:
        return self.pages.shape[0]

    @property
    def used_pages(self) -> int:
        n = c_int32()
        _check(self._lib.mi_prompt_cache_used(self._h, ctypes.byref(n), None))
        return n.value

    # -- attention -----------------------------------------------------------------
    def attention(self, entry: int, layer: int, q, k=None, v=None, cu_q=None, cu_k=None, causal: bool = True,
                  scale: float | None = None, out=None):
        """Attention of packed texts behind the prompt `entry`, with layer `layer`'s keys and values.

        q [tokens, n_heads, head_dim]; k, v [keys, n_kv_heads, head_dim], the texts' own (None: they have none); cu_q, cu_k
        int32 [texts + 1] on the device, where text i holds the queries cu_q[i] .. cu_q[i + 1] and the keys cu_k[i] ..
        cu_k[i + 1] (cu_k None: the same as cu_q; both None: one text).  With more keys than queries the first keys are the
        text's past: one query per text is the form for single tokens.  Every query sees the whole prompt; `causal`: of its
        own text the keys up to itself, otherwise all.  A query that sees nothing gets zeros.  scale: 1 / sqrt(head_dim) if
        None.  out: written in place if given (tokens of no text, in front of the first or behind the last, keep what they
        hold; in a new output they are zeros).  Inference only: no gradient."""
        import torch
        hd, kv, dtype, device = self.head_dim, self.n_kv_heads, self.dtype, self.device
        if entry >> 31 or layer >> 31:
            raise RuntimeError(f"mi_prompt_cache: prompt attention: no entry {entry}, layer {layer}")
        if q.dim() != 3 or q.shape[2] != hd:
            raise ValueError(f"PromptCache.attention: q [tokens, heads, {hd}], got {tuple(q.shape)}")
        if (k is None) != (v is None):
            raise ValueError("PromptCache.attention: k and v come together")
        if (torch.is_grad_enabled() and (q.requires_grad or (k is not None and (k.requires_grad or v.requires_grad)) or (out is not None and out.requires_grad))
                or getattr(torch.autograd.forward_ad, "_current_level", 0) >= 0):
            _no_gradient("attention", q, k, v, out)
        qs = q.stride()                              # (is_contiguous() does not look at the strides of axes of length 1)
        if q.dtype != dtype or q.device != device or qs[2] != 1 or (qs[0] | qs[1]) & 7 or q.data_ptr() & 15:
            q = self._fit(q, "q")
            qs = q.stride()
        tokens, heads, _ = q.shape
        if k is None:
            keys, kp, vp, ks, vs = 0, 0, 0, (0, 0), (0, 0)
        else:
            if k.dim() != 3 or k.shape != v.shape or k.shape[1] != kv or k.shape[2] != hd:
                raise ValueError(f"PromptCache.attention: k and v [keys, {kv}, {hd}], got {tuple(k.shape)} and {tuple(v.shape)}")
            k, v = self._fit(k, "k"), self._fit(v, "v")
            keys, kp, vp, ks, vs = k.shape[0], k.data_ptr(), v.data_ptr(), k.stride(), v.stride()
        if cu_q is None:
            if cu_k is not None:
                raise ValueError("PromptCache.attention: cu_k without cu_q")
            texts, cq, ck = 1, 0, 0
        else:
            if cu_k is None:
                if keys not in (0, tokens):
                    raise ValueError(f"PromptCache.attention: {keys} keys for {tokens} tokens need cu_k")
                cu_k = cu_q
            for cu in (cu_q, cu_k):
                if cu.dtype != torch.int32 or cu.dim() != 1 or cu.shape != cu_q.shape or cu.device != device or not cu.is_contiguous():
                    raise ValueError(f"PromptCache.attention: cu_q and cu_k are contiguous int32 [texts + 1] on {device}")
            texts, cq, ck = cu_q.shape[0] - 1, cu_q.data_ptr(), cu_k.data_ptr()
            if texts < 1:
                raise ValueError("PromptCache.attention: no text")
        rest = out is None
        if rest:
            out = q.new_empty((tokens, heads, hd))
            os = (heads * hd, hd)
        else:
            if out.dtype != dtype or out.device != device or out.shape != q.shape:
                raise ValueError(f"PromptCache.attention: out {tuple(q.shape)} {dtype} on {device}, got {tuple(out.shape)} {out.dtype} on {out.device}")
            os = out.stride()
            os = (os[0] if tokens > 1 else 0, os[1] if heads > 1 else 0, os[2])
            if os[2] != 1 or (os[0] | os[1]) & 7 or out.data_ptr() & 15:
                raise ValueError(f"PromptCache.attention: out with 16-byte aligned rows, got strides {out.stride()}")
            if tokens > 1 and os[0] == 0 or heads > 1 and os[1] == 0:
                raise ValueError("PromptCache.attention: out is broadcast: several of its rows are the same memory")
        if scale is None:
            scale = hd ** -0.5
        elif not 0 <= scale < math.inf:
            raise ValueError(f"PromptCache.attention: scale must be finite and not negative, got {scale}")
        head = (entry, layer, heads, tokens, keys, texts, q.data_ptr(), kp, vp, out.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1],
                cq, ck, causal, scale, rest, 0)
        shape, plans = (entry, heads, tokens, keys, texts), self._plans
        need = plans.get(shape)
        if need is None:
            need = self._workspace(head)
            if len(plans) > 1000:
                plans.clear()
            plans[shape] = need
        while True:
            ws = q.new_empty((need,), dtype=torch.uint8) if need else None
            if not self._lib.mi_prompt_attention(self._h, _ATTN.pack(*head, ws.data_ptr() if need else 0, need), self._stream()):
                if not rest:
                    torch.autograd.graph.increment_version(out)    # (a backward pass that saved it has to notice)
                return out
            why, had = self._lib.mi_enc_last_error().decode(), need
            need = self._workspace(head)
            if need <= had:                          # (else another thread has made the prompt longer in between)
                raise RuntimeError("mi_prompt_cache: " + why)

    def _workspace(self, head) -> int:
        n = c_int64()
        _check(self._lib.mi_prompt_attention_workspace(self._h, _ATTN.pack(*head, 0, 0), ctypes.byref(n)))
        return n.value
