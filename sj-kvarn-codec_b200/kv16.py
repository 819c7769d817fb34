"""Layers kept at 16 bits beside the sealed ones, over torch tensors: what goes from a projection to the cache (Qkv:
norm of every head, rotary positions, cache write, in one launch), the paged cache and the attention of one new token
that reads it (Cache), and who owns the pages (Pages: fork, extend with copy on write, free, compact).

    rope = kv16.Rope(128, base=1e6)
    cache = kv16.Cache.alloc(n_layers, n_pages, page, n_head_kv, head_dim, torch.bfloat16, n_rows, stride)
    pages = cache.pages()
    step = kv16.Qkv(head_dim, rope=rope, q_norm=wq, k_norm=wk, cache=cache)
    ...
    pages.extend(rows, lens, 1)                       # a page where the next position needs one, split where shared
    step(q, k, v, lens, q_out=q2, rows=rows, layer=il)  # position lens[i] of table row rows[i]
    out = cache.attend(il, q2, lens + 1, scale, rows=rows)

Calls run on the tensors' device, on torch's current stream there, and do not synchronise; tensors of another device raise
ValueError. Threads may share an object (a call of one waits for that of another until it is launched); what they launch on
several streams is theirs to order. Lengths, positions and row lists are int32 CUDA tensors, read when the kernels run;
sjk.lib().sjk_device_status() reports entries that pointed outside their arrays.
"""
import ctypes as C
import threading

import torch

import sjk

F32, F16, BF16 = 0, 1, 2
_TYPE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
_I32 = torch.int32
LAYOUTS = {"half": 0, "pair": 1}
SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}
NO_BLOCK = -1                                    # SJKVARN_NO_BLOCK in an int32 table

_L = None


def _lib():
    global _L
    if _L is None:
        _L = sjk.lib()
    return _L


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device):
    """torch's current stream of a device index, as a number."""
    return _raw_stream(device) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


_capturing = getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(device, call, *args):
    """call(*args) with `device` current: kernels, and limits set for them, go to the device that is."""
    if _current_device() == device:
        return call(*args)
    with torch.cuda.device(device):
        return call(*args)


def _list(t, what, device, n=None):
    """Address of an int32 vector on device `device` (None passes)."""
    if t is None:
        return None
    if t.dtype is not _I32 or t.dim() != 1 or t.get_device() != device or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise ValueError(f"{what}: an int32 vector" + (f" of {n} values" if n is not None else "") + f" on cuda:{device}")
    return t.data_ptr()


class _Rows:
    """A sjk_rows filled from [n][heads][D] tensors; a tensor of the last one's shape, strides and type changes the
    pointer only."""

    def __init__(self, c, what, D):
        self.c, self.what, self.D, self.like, self.n = c, what, D, None, -1

    def set(self, t, n, device):
        c = self.c
        if t is None:
            if self.like is not None:
                c.p, self.like = None, None
            return
        shape = t.shape
        like = (shape, t.stride(), t.dtype)
        if like != self.like or self.n != n:
            if len(shape) != 3 or shape[0] != n or shape[2] != self.D or like[1][2] != 1 or t.dtype not in _TYPE:
                raise ValueError(f"{self.what}: a CUDA tensor [{n}][heads][{self.D}] of 16- or 32-bit floats, channels adjacent")
            c.row_stride, c.head_stride, c.n_head, c.type = like[1][0], like[1][1], shape[1], _TYPE[t.dtype]
            self.like, self.n = like, n
        if t.get_device() != device:
            raise ValueError(f"{self.what}: a tensor on cuda:{device}")
        c.p = t.data_ptr()


class Rope:
    """Rotary positions of the first n_rot channels of a head (include/sjk.h, sjk_rope_config), for tensors of `device`
    (None: the current one)."""

    def __init__(self, n_rot, layout="half", base=10000.0, scaling="none", factor=1.0, n_ctx=0, beta_fast=32.0,
                 beta_slow=1.0, low=1.0, high=4.0, amp=0.0, device=None):
        self.cfg = sjk.RopeConfig(n_rot, LAYOUTS[layout], SCALINGS[scaling], base, factor, n_ctx, beta_fast, beta_slow,
                                  low, high, amp)
        self.c = sjk.RopeC()
        at = torch.device(device).index if isinstance(device, (str, torch.device)) else device
        self.device = _current_device() if at is None else at
        sjk.check(_launch(self.device, _lib().sjk_rope_init, C.byref(self.c), C.byref(self.cfg)), "rope_init")

    def __del__(self):
        if getattr(self, "c", None) is not None and _L is not None:
            _L.sjk_rope_free(C.byref(self.c))


def rope_steps(n_rot, layout="half", base=10000.0, scaling="none", factor=1.0, n_ctx=0, beta_fast=32.0, beta_slow=1.0,
               low=1.0, high=4.0, amp=0.0):
    """The table of a Rope on the host: (turns per position in units of 2^-64, amplitude). Needs no GPU."""
    cfg = sjk.RopeConfig(n_rot, LAYOUTS[layout], SCALINGS[scaling], base, factor, n_ctx, beta_fast, beta_slow, low, high, amp)
    step, a = (C.c_uint64 * 256)(), C.c_float()
    sjk.check(_lib().sjk_rope_steps(C.byref(cfg), step, C.byref(a)), "rope_steps")
    return list(step[: n_rot // 2]), a.value


class Pages:
    """Owner ledger of the pages behind `tables` (int32 [rows][stride], NO_BLOCK = no page) and `slabs` (CUDA tensors
    [layers][pages][...], contiguous within a page). ids, n_free: an existing stack of free ids (a value per page, of which
    the first n_free are free pages; pages that tables hold are not among them); without them every page is free."""

    def __init__(self, tables, page_tokens, slabs=(), n_pages=None, ids=None, n_free=None):
        if tables.dtype != torch.int32 or not tables.is_cuda or tables.dim() != 2 or not tables.is_contiguous():
            raise ValueError("tables: a contiguous int32 CUDA tensor [rows][stride]")
        n = slabs[0].shape[1] if n_pages is None else n_pages
        self.tables, self.slabs = tables, list(slabs)
        self._buf = torch.empty((_lib().sjk_pages_bytes(n) + 3) // 4, dtype=torch.int32, device=tables.device)
        self.c = c = sjk.PagesC(self._buf.data_ptr(), tables.data_ptr(), n, tables.shape[0], tables.shape[1], page_tokens)
        if len(self.slabs) > 4:
            raise ValueError("slabs: at most 4")
        if ids is not None and tuple(ids.shape) != (n,):
            raise ValueError(f"ids: {n} values, the first n_free of them free pages")
        free = n if n_free is None else int(n_free)
        if not 0 <= free <= n:
            raise ValueError(f"n_free: 0 to {n}")
        self._dev = tables.get_device()
        c.n_slabs = len(self.slabs)
        for i, s in enumerate(self.slabs):
            if s.get_device() != self._dev or s.dim() < 3 or s.shape[1] != n or not s[0].is_contiguous():
                raise ValueError("slabs: CUDA tensors [layers][pages][...] on the tables' device, pages of a layer contiguous")
            size = s.element_size()
            c.slabs[i] = sjk.Slab(s.data_ptr(), s.stride(1) * size, s.stride(0) * size, s.shape[0])
        self._c, self._L = C.byref(c), _lib()
        sjk.check(_launch(self._dev, self._L.sjk_pages_init, self._c, _stream(self._dev)), "pages_init")
        # what the last fork, extend and compact call reported (each overwritten by the next of its kind)
        self._forked = torch.zeros(1024, dtype=torch.int32, device=tables.device)
        self._extended = torch.zeros(1, dtype=torch.int32, device=tables.device)
        self._compacted = torch.zeros(2, dtype=torch.int32, device=tables.device)
        self.n_free, self.ids = self._buf[0:1], self._buf[4:4 + n]
        at = (self._L.sjk_pages_shares(self._c) - self._buf.data_ptr()) // 4
        self.shares = self._buf[at:at + n]
        if ids is not None:
            self.ids.copy_(ids)
            self.n_free.fill_(free)

    def fork(self, src, dst):
        """Rows dst get the pages of rows src, shared. Returns the device status vector (0, or a status code each)."""
        n = src.shape[0]
        st = self._forked if n <= 1024 else torch.empty(n, dtype=torch.int32, device=src.device)
        dev = self._dev
        rc = _launch(dev, self._L.sjk_pages_fork, self._c, _list(src, "src", dev), _list(dst, "dst", dev, n), n, st.data_ptr(), _stream(dev))
        if rc:
            raise sjk.SjkError(rc, "pages_fork")
        return st[:n]

    def extend(self, rows, lens, add=1):
        """Pages for the positions [lens, lens + add) of the rows, copied where shared; add: a number or a vector.
        Returns the device status (one value: 0, or why nothing was done)."""
        n = rows.shape[0]
        vec = isinstance(add, torch.Tensor)
        dev = self._dev
        rc = _launch(dev, self._L.sjk_pages_extend, self._c, _list(rows, "rows", dev), _list(lens, "lens", dev, n),
                     _list(add, "add", dev, n) if vec else None, 0 if vec else add, n, self._extended.data_ptr(), _stream(dev))
        if rc:
            raise sjk.SjkError(rc, "pages_extend")
        return self._extended

    def free(self, rows, first=None, end=None):
        """Entries [first, end) of the rows give their pages up (vectors; None: all)."""
        n = rows.shape[0]
        dev = self._dev
        rc = _launch(dev, self._L.sjk_pages_free, self._c, _list(rows, "rows", dev), _list(first, "first", dev, n), _list(end, "end", dev, n), n,
                     _stream(dev))
        if rc:
            raise sjk.SjkError(rc, "pages_free")

    def compact(self):
        """Used pages to the lowest ids. Returns a device vector: used pages, moved ones."""
        rc = _launch(self._dev, self._L.sjk_pages_compact, self._c, self._compacted.data_ptr(), _stream(self._dev))
        if rc:
            raise sjk.SjkError(rc, "pages_compact")
        return self._compacted

    def copy(self, src, dst):
        """Contents of pages src to pages dst, every layer of every slab."""
        n = src.shape[0]
        dev = self._dev
        rc = _launch(dev, self._L.sjk_pages_copy, self._c, _list(src, "src", dev), _list(dst, "dst", dev, n), n, _stream(dev))
        if rc:
            raise sjk.SjkError(rc, "pages_copy")


class Cache:
    """Paged 16-bit cache: k, v [layers][pages][page tokens][KV heads][D] of one 16-bit type and strides (any order of
    strides with adjacent channels), tables int32 [rows][stride]."""

    def __init__(self, k, v, tables):
        if k.dim() != 5 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.stride(4) != 1 or \
                k.dtype not in (torch.float16, torch.bfloat16) or not k.is_cuda or v.get_device() != k.get_device():
            raise ValueError("k, v: 16-bit tensors [layers][pages][tokens][heads][D] of one GPU with the same strides, channels adjacent")
        if tables.dtype != torch.int32 or tables.get_device() != k.get_device() or tables.dim() != 2 or not tables.is_contiguous():
            raise ValueError("tables: a contiguous int32 tensor [rows][stride] on the GPU of k and v")
        self.k, self.v, self.tables = k, v, tables
        n_layers, n_pages, page, H, D = k.shape
        st = k.stride()
        self.page_tokens, self.n_head_kv, self.head_dim = page, H, D
        self.layers = [sjk.Kv16(k[i].data_ptr(), v[i].data_ptr(), st[1], st[2], st[3], _TYPE[k.dtype], D, H, page, n_pages,
                                tables.data_ptr(), tables.shape[0], tables.shape[1]) for i in range(n_layers)]
        self._refs = [C.byref(x) for x in self.layers]
        self._q, self._o = _Rows(sjk.Rows(), "q", D), _Rows(sjk.Rows(), "out", D)
        self._qo = C.byref(self._q.c), C.byref(self._o.c)
        self._dev, self._L = k.get_device(), _lib()
        self._lock = threading.Lock()
        self._scratch = {}                       # by stream and number of query heads: calls of one stream follow one another

    @classmethod
    def alloc(cls, n_layers, n_pages, page_tokens, n_head_kv, head_dim, dtype, n_rows, stride, device="cuda"):
        shape = (n_layers, n_pages, page_tokens, n_head_kv, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                   torch.full((n_rows, stride), NO_BLOCK, dtype=torch.int32, device=device))

    def pages(self, ids=None, n_free=None):
        """A ledger over this cache's pages."""
        return Pages(self.tables, self.page_tokens, slabs=[self.k, self.v], ids=ids, n_free=n_free)

    def scratch_bytes(self, heads):
        """Bytes of scratch that attend needs for queries of so many heads."""
        size = self._L.sjk_kv16_attend_scratch_bytes(self._refs[0], heads)
        if not size:
            raise ValueError(f"{heads} query heads over {self.n_head_kv} heads of {self.head_dim} channels")
        return size

    def _scratch_of(self, st, q):
        """(tensor, address, bytes) for a call on stream st of the current device."""
        key, captured = (st, q.shape[1]), _capturing()
        scratch = None if captured else self._scratch.get(key)
        if scratch is None:
            size = self._L.sjk_kv16_attend_scratch_bytes(self._refs[0], q.shape[1])
            buf = torch.empty(size, dtype=torch.uint8, device=q.device)
            scratch = buf, buf.data_ptr(), size
            if not captured:
                self._scratch[key] = scratch
        return scratch

    def attend(self, layer, q, lens, scale, window=0, rows=None, out=None, scratch=None):
        """Attention of one new token per sequence: q [n][heads][D], lens int32 [n] (the newest position included), rows
        int32 [n] (None: sequence i is table row i). Returns out (q's type unless given).

        scratch: a uint8 tensor of scratch_bytes(heads) bytes that no overlapping call uses. None: the cache's own for the
        current stream, whose calls follow one another; while torch captures the stream, memory of the capture's pool, since
        graphs captured on one stream may be replayed on several. (Captured by other means than torch's: give it.)"""
        n, dev = q.shape[0], self._dev
        if _current_device() != dev:
            with torch.cuda.device(dev):
                return self.attend(layer, q, lens, scale, window, rows, out, scratch)
        if out is None:
            out = torch.empty_like(q)
        with self._lock:                         # the structs are the object's, and the call reads them without the interpreter's lock
            self._q.set(q, n, dev)
            self._o.set(out, n, dev)
            if n == 0:
                return out
            st = _stream(dev)
            if scratch is None:
                buf, address, size = self._scratch_of(st, q)
            elif scratch.dtype is torch.uint8 and scratch.is_contiguous() and scratch.get_device() == dev:
                address, size = scratch.data_ptr(), scratch.numel()
            else:
                raise ValueError(f"scratch: a contiguous uint8 tensor on cuda:{dev}")
            rc = self._L.sjk_kv16_attend(self._refs[layer], self._qo[0], _list(lens, "lens", dev, n), _list(rows, "rows", dev, n), n, scale,
                                         window, self._qo[1], address, size, st)
        if rc:
            raise sjk.SjkError(rc, "kv16_attend")
        return out


class Qkv:
    """From a projection's heads to cache rows in one launch: RMS norm of the query and key heads (weights q_norm,
    k_norm; None: none), rotary positions, and the write of K and V into `cache` and / or into row tensors."""

    def __init__(self, head_dim, rope=None, q_norm=None, k_norm=None, norm_bias=0.0, eps=1e-6, cache=None):
        self.head_dim, self.rope, self.cache = head_dim, rope, cache
        self._keep = (q_norm, k_norm)
        self._a = a = sjk.QkvArgs()
        a.head_dim, a.norm_bias, a.eps = head_dim, norm_bias, eps
        kinds = {w.dtype for w in self._keep if w is not None}
        for w in self._keep:
            if w is not None and (w.shape != (head_dim,) or not w.is_cuda or not w.is_contiguous() or w.dtype not in _TYPE):
                raise ValueError(f"norm weights: CUDA vectors of {head_dim} floats")
        if len(kinds) > 1:
            raise ValueError("norm weights: one type for both")
        a.q_norm, a.k_norm = (w.data_ptr() if w is not None else None for w in self._keep)
        a.norm_type = _TYPE[kinds.pop()] if kinds else F32
        if rope is not None:
            a.rope = rope.c
        at = {w.get_device() for w in self._keep if w is not None} | ({rope.device} if rope is not None else set()) | \
            ({cache._dev} if cache is not None else set())
        if len(at) > 1:
            raise ValueError("rope, norm weights and cache: of one GPU")
        self._dev = at.pop() if at else None
        self._ref, self._L = C.byref(a), _lib()
        self._layer = None
        self._lock = threading.Lock()
        # (the struct's own fields: setting them sets the struct's)
        self._rows = [_Rows(getattr(a, f), f, head_dim) for f in ("q", "k", "v", "q_out", "k_out", "v_out")]

    def __call__(self, q=None, k=None, v=None, pos=None, q_out=None, k_out=None, v_out=None, layer=0, rows=None, to_cache=True):
        """q, k, v: [n][heads][D] (views of one projection's rows are fine); pos int32 [n], a negative one is padding;
        rows int32 [n]: table row of every token (None: token i is row i). K and V go to the cache's layer unless
        to_cache is false; row outputs go where given (an input's own rows too)."""
        a = self._a
        some = q if q is not None else k if k is not None else v
        n, dev = some.shape[0], some.get_device()
        if dev < 0 or (self._dev is not None and dev != self._dev):
            raise ValueError("q, k, v: CUDA tensors" + (f" on cuda:{self._dev}" if self._dev is not None else ""))
        with self._lock:                         # the struct is the object's, and the call reads it without the interpreter's lock
            for r, t in zip(self._rows, (q, k, v, q_out, k_out, v_out)):
                r.set(t, n, dev)
            a.n_tok = n
            a.pos = _list(pos, "pos", dev, n)
            a.rows = _list(rows, "rows", dev, n)
            if n == 0:                           # empty tensors have no address
                return
            at = layer if self.cache is not None and to_cache else None
            if at != self._layer:
                a.cache = self.cache.layers[at] if at is not None else sjk.Kv16()
                self._layer = at
            rc = _launch(dev, self._L.sjk_qkv, self._ref, _stream(dev))
        if rc:
            raise sjk.SjkError(rc, "qkv")
