"""Rows after a prompt: a paged cache of keys and values, the attention of new rows over it, and the residual add between
two norms -- o1_kv_write, o1_kv_read, o1_kv_attention and o1_residual_norm on torch tensors.

Like every entry point they enqueue on the library's current stream (use_torch_stream()) and return at once.  Arguments that
do not fit raise O1Error; a slot, page or length that does not fit is found on the device (lib.o1_device_error() gives 70 or 71).
"""
import ctypes as C

import torch

from . import HEAD_DIM, KV_HEADS, KvCacheC, O1Error, check, lib

KINDS = {"bf16": (0, torch.bfloat16), "fp8": (1, torch.float8_e4m3fn), "int8": (2, torch.int8)}
_BY_DTYPE = {d: n for n, d in KINDS.values()}
BF16, I32, I64, F32 = torch.bfloat16, torch.int32, torch.int64, torch.float32


def _need(ok, what):
    if not ok:
        raise O1Error(what)


def _rows(t, heads, what):
    """Row pitch of bf16 rows [n, heads, 128] whose heads lie side by side."""
    if t.dtype is not BF16 or t.dim() != 3 or t.size(1) != heads or t.size(2) != HEAD_DIM:
        raise O1Error(f"{what}: bf16 [rows, {heads}, {HEAD_DIM}] wanted, got {t.dtype} {tuple(t.shape)}")
    ld, hs, cs = t.stride()
    if cs != 1 or (hs != HEAD_DIM and heads > 1) or not t.is_cuda:
        raise O1Error(f"{what}: a CUDA tensor with a row's heads side by side wanted, got strides {t.stride()}")
    return ld if t.size(0) > 1 else heads * HEAD_DIM


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
        if slots.dtype is not I64 or slots.dim() != 1 or not slots.is_contiguous() or slots.device != self.device:
            raise O1Error(f"{what}: slots int64 [rows], contiguous, on the cache's GPU wanted")
        return slots.size(0)

    def write(self, k, v, slots):
        """Rows k, v [n, kv_heads, 128] bf16 into slots [n] (int64, all different; negative: left out), quantised on the way."""
        n = self._slots(slots, "KvCache.write")
        ldk, ldv = _rows(k, self.kv_heads, "KvCache.write: k"), _rows(v, self.kv_heads, "KvCache.write: v")
        if k.size(0) != n or v.size(0) != n:
            raise O1Error("KvCache.write: k, v and slots differ in rows")
        rc = lib.o1_kv_write(self._ref, k.data_ptr(), ldk, v.data_ptr(), ldv, slots.data_ptr(), n)
        if rc:
            check(rc, "o1_kv_write")

    def read(self, slots, out=None):
        """(k, v) [n, kv_heads, 128] bf16 of slots [n]; zeros where a slot is negative.  out: a pair of tensors to fill, rows of any pitch."""
        n = self._slots(slots, "KvCache.read")
        if out is None:
            both = torch.empty(2, n, self.kv_heads, HEAD_DIM, dtype=BF16, device=self.device)
            k, v = both[0], both[1]
            ldk = ldv = self.kv_heads * HEAD_DIM
        else:
            k, v = out
            ldk, ldv = _rows(k, self.kv_heads, "KvCache.read: k"), _rows(v, self.kv_heads, "KvCache.read: v")
            if k.size(0) != n or v.size(0) != n:
                raise O1Error("KvCache.read: out and slots differ in rows")
        rc = lib.o1_kv_read(self._ref, k.data_ptr(), ldk, v.data_ptr(), ldv, slots.data_ptr(), n)
        if rc:
            check(rc, "o1_kv_read")
        return k, v

    def workspace(self, heads):
        """Scratch of attend(): one for each stream the calls run on, as calls that overlap must not share it."""
        key = (lib.o1_get_stream(), heads)
        w = self._work.get(key)
        if w is None:
            need = lib.o1_kv_attention_workspace_bytes(heads, self.kv_heads)
            _need(need >= 0, f"KvCache.attend: heads {heads} (a multiple of kv_heads {self.kv_heads})")
            w = self._work[key] = torch.zeros(need, dtype=torch.uint8, device=self.device)
        return w

    def attend(self, q, pages, lens, k=None, v=None, out=None, lse=None, scale=None):
        """Attention of one new row per sequence, q [batch, heads, 128] bf16, over its first lens[b] cached rows.

        pages [batch, width] int32: the pages of each sequence in order (entries behind its last page are not read); lens [batch] int32.
        k, v [batch, kv_heads, 128]: each sequence's row at position lens[b] - 1, stored into the cache and attended to.
        Returns out [batch, heads, 128] bf16, with lse=True (or a tensor [batch, heads] fp32) a pair (out, log-sum-exp).  An empty sequence
        gives zeros and -inf.  scale: 1 / sqrt(128)."""
        if q.dim() != 3:
            raise O1Error("KvCache.attend: q [batch, heads, 128] wanted")
        n, heads = q.size(0), q.size(1)
        ldq = _rows(q, heads, "KvCache.attend: q")
        if pages.dtype is not I32 or pages.dim() != 2 or pages.size(0) != n or pages.stride(1) != 1 or pages.device != self.device:
            raise O1Error("KvCache.attend: pages int32 [batch, width] on the cache's GPU wanted")
        if lens.dtype is not I32 or lens.dim() != 1 or lens.size(0) != n or not lens.is_contiguous() or lens.device != self.device:
            raise O1Error("KvCache.attend: lens int32 [batch] on the cache's GPU wanted")
        pk = pv = None
        ldk = ldv = 0
        if k is not None or v is not None:
            if k is None or v is None or k.size(0) != n or v.size(0) != n:
                raise O1Error("KvCache.attend: k and v [batch, kv_heads, 128], both or neither")
            ldk, ldv = _rows(k, self.kv_heads, "KvCache.attend: k"), _rows(v, self.kv_heads, "KvCache.attend: v")
            pk, pv = k.data_ptr(), v.data_ptr()
        if out is None:
            out = torch.empty(n, heads, HEAD_DIM, dtype=BF16, device=self.device)
            ldo = heads * HEAD_DIM
        else:
            ldo = _rows(out, heads, "KvCache.attend: out")
            if out.size(0) != n:
                raise O1Error("KvCache.attend: out and q differ in rows")
        if lse is True:
            lse = torch.empty(n, heads, dtype=F32, device=self.device)
        elif lse is False:
            lse = None
        elif lse is not None and (lse.dtype is not F32 or tuple(lse.shape) != (n, heads) or not lse.is_contiguous()):
            raise O1Error("KvCache.attend: lse fp32 [batch, heads] wanted")
        w = self.workspace(heads)
        rc = lib.o1_kv_attention(self._ref, q.data_ptr(), ldq, pk, ldk, pv, ldv, pages.data_ptr(), pages.stride(0) if n > 1 else pages.size(1),
                                 pages.size(1), lens.data_ptr(), out.data_ptr(), ldo, None if lse is None else lse.data_ptr(), n, heads,
                                 HEAD_DIM ** -0.5 if scale is None else scale, w.data_ptr(), w.numel())
        if rc:
            check(rc, "o1_kv_attention")
        return out if lse is None else (out, lse)


def residual_norm(x, branch, pre_w, post_w=None, gate=None, scale=None, shift=None, alpha=1.0, eps=1e-6, y=None, h=None):
    """(y, h): y = x + alpha * gate * u with u = branch, or rmsnorm(branch) * post_w; h = rmsnorm(y) * pre_w, and * (1 + scale) + shift.

    x, branch [rows, cols] bf16 with rows of any pitch; the weights [cols]; gate, scale, shift [cols] or [groups, cols], a vector for each
    rows / groups rows.  pre_w None: no norm behind the sum, h is None.  y, h: tensors to fill (y may be x or branch)."""
    if x.dtype is not BF16 or x.dim() != 2 or not x.is_cuda or branch.dtype is not BF16 or branch.shape != x.shape or not branch.is_cuda:
        raise O1Error("residual_norm: x and branch bf16 [rows, cols] on the GPU wanted")
    rows, cols = x.shape
    groups = 1
    p = []
    for name, t, many in (("post_w", post_w, False), ("gate", gate, True), ("pre_w", pre_w, False), ("scale", scale, True), ("shift", shift, True)):
        if t is None:
            p.append(None)
            continue
        if t.dtype is not BF16 or t.size(-1) != cols or not t.is_contiguous() or not t.is_cuda or t.dim() > (2 if many else 1):
            raise O1Error(f"residual_norm: {name} bf16 [{'groups, ' if many else ''}{cols}] wanted")
        if many:
            g = t.size(0) if t.dim() == 2 else 1
            if g != groups and groups != 1 and g != 1 or g == 0:
                raise O1Error("residual_norm: gate, scale and shift differ in groups")
            groups = max(groups, g)
        p.append(t)
    if groups > 1:
        for i in (1, 3, 4):
            if p[i] is not None and (p[i].dim() == 1 or p[i].size(0) == 1):
                p[i] = p[i].reshape(1, cols).expand(groups, cols).contiguous()
    if y is None:
        y = torch.empty(rows, cols, dtype=BF16, device=x.device)
    if h is None and pre_w is not None:
        h = torch.empty(rows, cols, dtype=BF16, device=x.device)
    for t in (y, h):
        if t is not None and (t.dtype is not BF16 or t.shape != x.shape or not t.is_cuda):
            raise O1Error("residual_norm: y and h bf16 [rows, cols] wanted")
    if pre_w is None and h is not None:
        raise O1Error("residual_norm: h without pre_w")
    ld = []
    for t in (x, branch, y, h):
        if t is not None and t.stride(1) != 1 and cols > 1:
            raise O1Error("residual_norm: the values of a row must lie side by side")
        ld.append(0 if t is None else t.stride(0) if rows > 1 else cols)
    a = [None if t is None else t.data_ptr() for t in p]
    rc = lib.o1_residual_norm(x.data_ptr(), ld[0], branch.data_ptr(), ld[1], a[0], a[1], alpha, a[2], a[3], a[4], groups, y.data_ptr(), ld[2],
                              None if h is None else h.data_ptr(), ld[3], rows, cols, eps)
    if rc:
        check(rc, "o1_residual_norm")
    return y, h
