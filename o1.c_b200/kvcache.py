"""Rows after a prompt: a paged cache of keys and values, the attention of new rows over it, the residual add between
two norms -- o1_kv_write, o1_kv_read, o1_kv_attention and o1_residual_norm on torch tensors -- and a Decoder that continues prompts with them.

Like every entry point they enqueue on the library's current stream (use_torch_stream()) and return at once.  Arguments that
do not fit raise O1Error; a slot, page or length that does not fit is found on the device (lib.o1_device_error() gives 70 or 71).
"""
import ctypes as C

import torch

from . import HEAD_DIM, KV_HEADS, KvCacheC, O1Error, check, lib, ptr

KINDS = {"bf16": (0, torch.bfloat16), "fp8": (1, torch.float8_e4m3fn), "int8": (2, torch.int8)}
_BY_DTYPE = {d: n for n, d in KINDS.values()}
BF16, I32, I64, F32 = torch.bfloat16, torch.int32, torch.int64, torch.float32
SCALE = HEAD_DIM ** -0.5
_write, _read, _attend, _norm, _stream = lib.o1_kv_write, lib.o1_kv_read, lib.o1_kv_attention, lib.o1_residual_norm, lib.o1_get_stream


def _need(ok, what):
    if not ok:
        raise O1Error(what)


def _rows(t, heads, what):
    """Rows and row pitch of bf16 rows [n, heads, 128] whose heads lie side by side.  (Short on purpose: for a few rows a call is bound by its checks.)"""
    shape = t.shape
    if t.dtype is not BF16 or len(shape) != 3 or shape[1] != heads or shape[2] != HEAD_DIM:
        raise O1Error(f"{what}: bf16 [rows, {heads}, {HEAD_DIM}] wanted, got {t.dtype} {tuple(shape)}")
    ld, hs, cs = t.stride()
    if cs != 1 or (hs != HEAD_DIM and heads > 1) or not t.is_cuda:
        raise O1Error(f"{what}: a CUDA tensor with a row's heads side by side wanted, got strides {t.stride()}")
    n = shape[0]
    return n, (ld if n > 1 else heads * HEAD_DIM)


class KvCache:
    """Keys and values of many sequences in pages of page_size tokens, [pages, kv_heads, page_size, 128].

    kind: "bf16", or "fp8" / "int8" (a byte a value and one fp32 scale for each token and head).  A token's slot is
    page * page_size + its place in the page; which pages a sequence has is the caller's table."""

    def __init__(self, pages, page_size=64, kind="bf16", kv_heads=KV_HEADS, device="cuda"):
        _need(kind in KINDS, f"KvCache: kind {kind!r} (one of {', '.join(KINDS)})")
        shape = (pages, kv_heads, page_size, HEAD_DIM)
        dtype = KINDS[kind][1]
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) if kind != "bf16" else
                torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        ks, vs = (torch.zeros(shape[:3], device=device) if kind != "bf16" else None for _ in range(2))
        self._set(k, v, ks, vs)

    @classmethod
    def over(cls, k, v, k_scale=None, v_scale=None):
        """A cache in tensors that the caller has."""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale)
        return self

    def _set(self, k, v, k_scale, v_scale):
        _need(k.dtype in _BY_DTYPE and k.dim() == 4 and k.size(3) == HEAD_DIM, "KvCache: k [pages, kv_heads, page_size, 128] bf16, float8_e4m3fn or int8 wanted")
        _need(v.dtype == k.dtype and v.shape == k.shape, "KvCache: v differs from k in shape or type")
        kind = _BY_DTYPE[k.dtype]
        tensors = [k, v]
        if kind:
            for s in (k_scale, v_scale):
                _need(s is not None and s.dtype is F32 and s.shape == k.shape[:3], "KvCache: scales [pages, kv_heads, page_size] fp32 wanted")
                tensors.append(s)
        for t in tensors:
            _need(t.is_cuda and t.device == k.device and t.is_contiguous() and t.data_ptr() % 16 == 0, "KvCache: contiguous, 16-byte aligned tensors of one GPU wanted")
        _need(k.size(0) > 0 and k.size(1) > 0 and k.size(2) > 0 and k.size(2) % 16 == 0, "KvCache: page_size must be a multiple of 16, pages and kv_heads positive")
        self.k, self.v, self.k_scale, self.v_scale = k, v, (k_scale if kind else None), (v_scale if kind else None)
        self.pages, self.kv_heads, self.page_size = k.size(0), k.size(1), k.size(2)
        self.device = k.device
        p = [t.data_ptr() for t in tensors] + ([] if kind else [None, None])
        self.c = KvCacheC(*p, kind, self.pages, self.page_size, self.kv_heads, HEAD_DIM)
        self._ref = C.byref(self.c)
        self._work = {}

    def _slots(self, slots, what):
        shape = slots.shape
        if slots.dtype is not I64 or len(shape) != 1 or not slots.is_contiguous() or slots.device != self.device:
            raise O1Error(f"{what}: slots int64 [rows], contiguous, on the cache's GPU wanted")
        return shape[0]

    def write(self, k, v, slots):
        """Rows k, v [n, kv_heads, 128] bf16 into slots [n] (int64, all different; negative: left out), quantised on the way."""
        n = self._slots(slots, "KvCache.write")
        nk, ldk = _rows(k, self.kv_heads, "KvCache.write: k")
        nv, ldv = _rows(v, self.kv_heads, "KvCache.write: v")
        if nk != n or nv != n:
            raise O1Error("KvCache.write: k, v and slots differ in rows")
        rc = _write(self._ref, k.data_ptr(), ldk, v.data_ptr(), ldv, slots.data_ptr(), n)
        if rc:
            check(rc, "o1_kv_write")

    def read(self, slots, out=None):
        """(k, v) [n, kv_heads, 128] bf16 of slots [n]; zeros where a slot is negative.  out: a pair of tensors to fill, rows of any pitch."""
        n = self._slots(slots, "KvCache.read")
        if out is None:
            k = torch.empty(n, self.kv_heads, HEAD_DIM, dtype=BF16, device=self.device)
            v = torch.empty_like(k)
            ldk = ldv = self.kv_heads * HEAD_DIM
        else:
            k, v = out
            nk, ldk = _rows(k, self.kv_heads, "KvCache.read: k")
            nv, ldv = _rows(v, self.kv_heads, "KvCache.read: v")
            if nk != n or nv != n:
                raise O1Error("KvCache.read: out and slots differ in rows")
        rc = _read(self._ref, k.data_ptr(), ldk, v.data_ptr(), ldv, slots.data_ptr(), n)
        if rc:
            check(rc, "o1_kv_read")
        return k, v

    def _workspace(self, heads):
        """Scratch of attend(), its address and bytes: one for each stream the calls run on, as calls that overlap must not share it."""
        need = lib.o1_kv_attention_workspace_bytes(heads, self.kv_heads)
        _need(need >= 0, f"KvCache.attend: heads {heads} (a multiple of kv_heads {self.kv_heads})")
        t = torch.zeros(need, dtype=torch.uint8, device=self.device)
        w = self._work[_stream(), heads] = (t.data_ptr(), need, t)
        return w

    def attend(self, q, pages, lens, k=None, v=None, out=None, lse=None, scale=None):
        """Attention of one new row per sequence, q [batch, heads, 128] bf16, over its first lens[b] cached rows.

        pages [batch, width] int32: the pages of each sequence in order (entries behind its last page are not read); lens [batch] int32.
        k, v [batch, kv_heads, 128]: each sequence's row at position lens[b] - 1, stored into the cache and attended to.
        Returns out [batch, heads, 128] bf16, with lse=True (or a tensor [batch, heads] fp32) a pair (out, log-sum-exp).  An empty sequence
        gives zeros and -inf.  scale: 1 / sqrt(128)."""
        shape = q.shape
        if len(shape) != 3:
            raise O1Error("KvCache.attend: q [batch, heads, 128] wanted")
        heads = shape[1]
        n, ldq = _rows(q, heads, "KvCache.attend: q")
        shape = pages.shape
        if pages.dtype is not I32 or len(shape) != 2 or shape[0] != n or pages.device != self.device:
            raise O1Error("KvCache.attend: pages int32 [batch, width] on the cache's GPU wanted")
        width = shape[1]
        ldp, cs = pages.stride()
        if cs != 1 and width > 1:
            raise O1Error("KvCache.attend: the pages of a sequence must lie side by side")
        shape = lens.shape
        if lens.dtype is not I32 or len(shape) != 1 or shape[0] != n or not lens.is_contiguous() or lens.device != self.device:
            raise O1Error("KvCache.attend: lens int32 [batch] on the cache's GPU wanted")
        pk = pv = pl = None
        ldk = ldv = 0
        if k is not None and v is not None:
            nk, ldk = _rows(k, self.kv_heads, "KvCache.attend: k")
            nv, ldv = _rows(v, self.kv_heads, "KvCache.attend: v")
            if nk != n or nv != n:
                raise O1Error("KvCache.attend: k, v and q differ in rows")
            pk, pv = k.data_ptr(), v.data_ptr()
        elif k is not None or v is not None:
            raise O1Error("KvCache.attend: k and v [batch, kv_heads, 128], both or neither")
        if out is None:
            out = torch.empty_like(q)
            ldo = out.stride()[0] if n > 1 else heads * HEAD_DIM
        else:
            no, ldo = _rows(out, heads, "KvCache.attend: out")
            if no != n:
                raise O1Error("KvCache.attend: out and q differ in rows")
        if lse is True:
            lse = torch.empty(n, heads, dtype=F32, device=self.device)
            pl = lse.data_ptr()
        elif lse is not None and lse is not False:
            if lse.dtype is not F32 or tuple(lse.shape) != (n, heads) or not lse.is_contiguous() or not lse.is_cuda:
                raise O1Error("KvCache.attend: lse fp32 [batch, heads] wanted")
            pl = lse.data_ptr()
        w = self._work.get((_stream(), heads)) or self._workspace(heads)
        rc = _attend(self._ref, q.data_ptr(), ldq, pk, ldk, pv, ldv, pages.data_ptr(), ldp if n > 1 else width, width, lens.data_ptr(),
                     out.data_ptr(), ldo, pl, n, heads, SCALE if scale is None else scale, w[0], w[1])
        if rc:
            check(rc, "o1_kv_attention")
        return out if pl is None else (out, lse)


def residual_norm(x, branch, pre_w, post_w=None, gate=None, scale=None, shift=None, alpha=1.0, eps=1e-6, y=None, h=None):
    """(y, h): y = x + alpha * gate * u with u = branch, or rmsnorm(branch) * post_w; h = rmsnorm(y) * pre_w, and * (1 + scale) + shift.

    x, branch [rows, cols] bf16 with rows of any pitch; the weights [cols]; gate, scale, shift [cols] or [groups, cols], a vector for each
    rows / groups rows.  pre_w None: no norm behind the sum, h is None.  y, h: tensors to fill (y may be x or branch)."""
    shape = x.shape
    if x.dtype is not BF16 or branch.dtype is not BF16 or len(shape) != 2 or branch.shape != shape or not x.is_cuda or not branch.is_cuda:
        raise O1Error("residual_norm: x and branch bf16 [rows, cols] on the GPU wanted")
    rows, cols = shape
    p_post = p_pre = p_gate = p_scale = p_shift = p_h = None
    groups, ldh = 1, 0
    if post_w is not None:
        _vector(post_w, cols, 1, "post_w")
        p_post = post_w.data_ptr()
    if gate is not None:
        groups = _vector(gate, cols, 2, "gate")
    if scale is not None:
        g = _vector(scale, cols, 2, "scale")
        groups = g if groups == 1 else groups
        _need(shift is not None, "residual_norm: scale without shift")
    if shift is not None:
        g = _vector(shift, cols, 2, "shift")
        groups = g if groups == 1 else groups
    if groups > 1:
        gate, scale, shift = (_each_group(t, cols, groups) for t in (gate, scale, shift))
    if gate is not None:
        p_gate = gate.data_ptr()
    if scale is not None:
        p_scale = scale.data_ptr()
    if shift is not None:
        p_shift = shift.data_ptr()
    if y is None:
        y = torch.empty_like(x)
    elif y.dtype is not BF16 or y.shape != shape or not y.is_cuda:
        raise O1Error("residual_norm: y bf16 [rows, cols] wanted")
    if pre_w is not None:
        _vector(pre_w, cols, 1, "pre_w")
        p_pre = pre_w.data_ptr()
        if h is None:
            h = torch.empty_like(x)
        elif h.dtype is not BF16 or h.shape != shape or not h.is_cuda:
            raise O1Error("residual_norm: h bf16 [rows, cols] wanted")
        ldh, ch = h.stride()
        p_h = h.data_ptr()
    elif h is not None:
        raise O1Error("residual_norm: h without pre_w")
    else:
        ch = 1
    (ldx, cx), (ldb, cb), (ldy, cy) = x.stride(), branch.stride(), y.stride()
    if not cx == cb == cy == ch == 1 and cols > 1:
        raise O1Error("residual_norm: the values of a row must lie side by side")
    if rows == 1 or cols == 1:
        ldx, ldb, ldy, ldh = (max(ld, cols) for ld in (ldx, ldb, ldy, ldh))
    rc = _norm(x.data_ptr(), ldx, branch.data_ptr(), ldb, p_post, p_gate, alpha, p_pre, p_scale, p_shift, groups, y.data_ptr(), ldy, p_h, ldh, rows, cols, eps)
    if rc:
        check(rc, "o1_residual_norm")
    return y, h


def _vector(t, cols, dims, name):
    """The number of vectors [cols] in t."""
    shape = t.shape
    if t.dtype is not BF16 or not 0 < len(shape) <= dims or shape[-1] != cols or not t.is_contiguous() or not t.is_cuda or shape[0] == 0:
        raise O1Error(f"residual_norm: {name} bf16 [{'groups, ' if dims > 1 else ''}{cols}] wanted")
    return shape[0] if len(shape) == 2 else 1


def _each_group(t, cols, groups):
    if t is None or t.numel() == groups * cols:
        return t
    _need(t.numel() == cols, "residual_norm: gate, scale and shift differ in groups")
    return t.reshape(1, cols).expand(groups, cols).contiguous()


class Decoder:
    """Continues prompts through the decoder blocks, a row of every sequence at a time, over cached keys and values.

    weights: Weights (or GgufWeights).  max_seqs sequences of at most max_tokens rows each; kind: how keys and values are kept (KvCache).
    prompt() and step() return rows behind the final norm, [rows, hidden] bf16, and enqueue on the library's current stream."""

    def __init__(self, weights, max_seqs, max_tokens, kind="bf16", page_size=64):
        d = weights.dims
        self.w, self.device = weights, weights.device
        self.dims = (d["heads"], d["kv_heads"], d["hidden"], d["ff"], d["head_dim"], d["vocab"])
        self.max_seqs, self.max_tokens, self.page_size = max_seqs, max_tokens, page_size
        self.width = -(-max_tokens // page_size)
        layers = weights.binding.n_layers
        self.caches = [KvCache(max_seqs * self.width, page_size, kind, d["kv_heads"], self.device) for _ in range(layers)]
        self._c = (KvCacheC * layers)(*[c.c for c in self.caches])
        self._free = list(range(max_seqs * self.width - 1, -1, -1))
        self._pages, self._len, self._table = {}, {}, {}
        self._next = 0
        self._scratch = {}

    def _room(self, rows):
        """Scratch for so many rows on the current stream."""
        key = _stream()
        s = self._scratch.get(key)
        need = lib.o1_decode_scratch_bytes(rows, *self.dims[:5])
        if s is None or s.numel() < need:
            s = self._scratch[key] = torch.zeros(need, dtype=torch.uint8, device=self.device)
        return s

    def _grow(self, seq, tokens):
        """Room for so many rows of the sequence; its pages' table on the GPU."""
        pages = self._pages[seq]
        if tokens > self.max_tokens:
            raise O1Error(f"Decoder: a sequence of {tokens} rows (max_tokens is {self.max_tokens})")
        while len(pages) * self.page_size < tokens:
            pages.append(self._free.pop())
            self._table[seq] = None
        if self._table[seq] is None:
            row = torch.zeros(self.width, dtype=torch.int32)
            row[:len(pages)] = torch.tensor(pages, dtype=torch.int32)
            self._table[seq] = row.to(self.device)

    def prompt(self, ids):
        """A new sequence of rows ids [n] (int64): (its name, hidden rows [n, hidden])."""
        n = ids.numel()
        if ids.dtype is not I64 or ids.dim() != 1 or n == 0 or not ids.is_cuda:
            raise O1Error("Decoder.prompt: ids int64 [n] on the GPU wanted, n > 0")
        if len(self._pages) == self.max_seqs:
            raise O1Error(f"Decoder.prompt: {self.max_seqs} sequences are open")
        seq = self._next
        self._pages[seq], self._len[seq], self._table[seq] = [], 0, None
        try:
            self._grow(seq, n)
        except O1Error:
            self.close(seq)
            raise
        self._next += 1
        self._len[seq] = n
        t = torch.arange(n, device=self.device)
        slots = self._table[seq].long()[t // self.page_size] * self.page_size + t % self.page_size
        pos = t.float().expand(3, n).contiguous()
        out = torch.empty(n, self.dims[2], dtype=BF16, device=self.device)
        s = self._room(n)
        check(lib.o1_prompt_rows(C.byref(self.w.binding), self._c, ptr(ids.contiguous()), ptr(pos), ptr(slots), ptr(s), s.numel(), ptr(out), n, *self.dims),
              "o1_prompt_rows")
        return seq, out

    def step(self, seqs, ids):
        """One new row of each sequence in seqs (all different), ids [len(seqs)] (int64): hidden rows [len(seqs), hidden]."""
        n = len(seqs)
        if ids.dtype is not I64 or ids.dim() != 1 or ids.numel() != n or not ids.is_cuda or len(set(seqs)) != n:
            raise O1Error("Decoder.step: ids int64, one for each of different sequences, on the GPU wanted")
        for s in seqs:
            if s not in self._pages:
                raise O1Error(f"Decoder.step: no sequence {s}")
            self._grow(s, self._len[s] + 1)
        for s in seqs:
            self._len[s] += 1
        lens = torch.tensor([self._len[s] for s in seqs], dtype=I32).to(self.device)
        pages = torch.stack([self._table[s] for s in seqs]) if n else torch.zeros(0, self.width, dtype=I32, device=self.device)
        pos = (lens - 1).float().expand(3, n).contiguous()
        out = torch.empty(n, self.dims[2], dtype=BF16, device=self.device)
        s = self._room(n)
        check(lib.o1_decode_step(C.byref(self.w.binding), self._c, ptr(ids.contiguous()), ptr(pos), ptr(pages), self.width, self.width, ptr(lens), ptr(s), s.numel(),
                                 ptr(out), n, *self.dims), "o1_decode_step")
        return out

    def rows(self, seq, layer):
        """(keys, values) [rows, kv_heads, 128] bf16 that a layer keeps of a sequence, as KvCache.read gives them."""
        if seq not in self._pages:
            raise O1Error(f"Decoder.rows: no sequence {seq}")
        t = torch.arange(self._len[seq], device=self.device)
        return self.caches[layer].read(self._table[seq].long()[t // self.page_size] * self.page_size + t % self.page_size)

    def close(self, seq):
        """Gives a sequence's pages back.  (Calls on other streams that still read them are the caller's to wait for.)"""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._len[seq], self._table[seq]
