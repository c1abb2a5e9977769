"""Rows after a prompt: a paged cache of keys and values, the attention of new rows over it, the residual add between
two norms -- o1_kv_write, o1_kv_read, o1_kv_attention and o1_residual_norm on torch tensors -- and a Decoder that continues prompts with them.

Like every entry point they enqueue on the library's current stream (use_torch_stream()) and return at once.  Arguments that
do not fit raise O1Error; a slot, page or length that does not fit is found on the device (lib.o1_device_error() gives 70 or 71).
Where torch's current stream is another one, what these calls make (caches, results, tables) is made, filled and freed in the order of the library's;
ordering that, and their inputs, with torch's own work is the caller's.
"""
import ctypes as C
import os

import torch

_BINDING = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_binding.so")
if not os.path.exists(_BINDING):
    raise ImportError(f"{_BINDING} is missing: build it with `python o1.c_b200/build.py`. There is no fallback path.")

from . import _binding  # noqa: E402

if _binding.torch_version != torch.__version__.split("+")[0]:
    raise ImportError(f"{_BINDING} is of torch {_binding.torch_version}, this is {torch.__version__}: build it with `python o1.c_b200/build.py`")

from . import HEAD_DIM, KV_HEADS, KvCacheC, O1Error, _on_library, check, lib, ptr  # noqa: E402

KINDS = {"bf16": (0, torch.bfloat16), "fp8": (1, torch.float8_e4m3fn), "int8": (2, torch.int8)}
_BY_DTYPE = {d: n for n, d in KINDS.values()}
BF16, I32, I64, F32 = torch.bfloat16, torch.int32, torch.int64, torch.float32
_stream = lib.o1_get_stream
_binding.setup(*(C.cast(f, C.c_void_p).value for f in (lib.o1_kv_write, lib.o1_kv_read, lib.o1_kv_attention, lib.o1_residual_norm, lib.o1_get_stream, lib.o1_capture_id)),
               O1Error, check)


def _need(ok, what):
    if not ok:
        raise O1Error(what)


def _zeros(n, device):
    """n bytes of zeros, filled on the library's current stream."""
    with _on_library(device):
        return torch.zeros(n, dtype=torch.uint8, device=device)


def _to_gpu(values, device):
    """A list of the host's as int32 on the GPU, copied on the library's current stream from pinned memory: the host does not wait for what is under way."""
    with _on_library(device):
        return torch.tensor(values, dtype=I32, pin_memory=True).to(device, non_blocking=True)


class _Workspace:
    """Scratch of attend(), for all caches: one for each device, stream and capture, as calls that overlap must not share it (and a capture's is filled by its graph).
    A stream's stays, a capture's goes when its graph has."""
    made, watched = {}, {}

    def __init__(self, device, nbytes):
        self.scratch = _zeros(nbytes, device)
        self.address = self.scratch.data_ptr()

    def data_ptr(self):
        return self.address

    @classmethod
    def get(cls, device, capture, nbytes):
        key = (device, _stream(), capture, nbytes)
        if key not in cls.made:
            for gone in [c for c in cls.watched if lib.o1_capture_gone(c)]:
                for k in cls.watched.pop(gone):
                    cls.made.pop(k).scratch = None
            cls.made[key] = cls(device, nbytes)
            if capture and (capture in cls.watched or lib.o1_capture_watch()):
                cls.watched.setdefault(capture, []).append(key)
        return cls.made[key]


class KvCache:
    """Keys and values of many sequences in pages of page_size tokens, [pages, kv_heads, page_size, 128].

    kind: "bf16", or "fp8" / "int8" (a byte a value and one fp32 scale for each token and head).  A token's slot is
    page * page_size + its place in the page; which pages a sequence has is the caller's table."""

    def __init__(self, pages, page_size=64, kind="bf16", kv_heads=KV_HEADS, device="cuda"):
        _need(kind in KINDS, f"KvCache: kind {kind!r} (one of {', '.join(KINDS)})")
        shape = (pages, kv_heads, page_size, HEAD_DIM)
        dtype = KINDS[kind][1]
        with _on_library(device):
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
        self._h = _binding.handle(C.addressof(self.c), self.kv_heads, k.get_device())
        self._work = {}

    def write(self, k, v, slots):
        """Rows k, v [n, kv_heads, 128] bf16 into slots [n] (int64, all different; negative: left out), quantised on the way."""
        _binding.write(self._h, k, v, slots)

    def read(self, slots, out=(None, None)):
        """(k, v) [n, kv_heads, 128] bf16 of slots [n]; zeros where a slot is negative.  out: a pair of tensors to fill, rows of any pitch."""
        return _binding.read(self._h, slots, *out)

    def _workspace(self, heads):
        """Address and bytes of attend()'s scratch for the library's current stream."""
        need = lib.o1_kv_attention_workspace_bytes(heads, self.kv_heads)
        _need(need >= 0, f"KvCache.attend: heads {heads} (a multiple of kv_heads {self.kv_heads})")
        capture = lib.o1_capture_id()
        w = _Workspace.get(self.device, capture, need)
        self._work = {k: old for k, old in self._work.items() if old.scratch is not None}
        self._work[_stream(), capture, heads] = w
        return w.address, need

    def attend(self, q, pages, lens, k=None, v=None, out=None, lse=None, scale=None):
        """Attention of one new row per sequence, q [batch, heads, 128] bf16, over its first lens[b] cached rows.

        pages [batch, width] int32: the pages of each sequence in order (entries behind its last page are not used); lens [batch] int32.
        k, v [batch, kv_heads, 128]: each sequence's row at position lens[b] - 1, stored into the cache and attended to.
        Returns out [batch, heads, 128] bf16, with lse=True (or a tensor [batch, heads] fp32) a pair (out, log-sum-exp).  An empty sequence
        gives zeros and -inf.  scale: 1 / sqrt(128)."""
        return _binding.attend(self._h, self, q, pages, lens, k, v, out, lse, scale)


def residual_norm(x, branch, pre_w, post_w=None, gate=None, scale=None, shift=None, alpha=1.0, eps=1e-6, y=None, h=None):
    """(y, h): y = x + alpha * gate * u with u = branch, or rmsnorm(branch) * post_w; h = rmsnorm(y) * pre_w, and * (1 + scale) + shift.

    x, branch [rows, cols] bf16 with rows of any pitch; the weights [cols]; gate, scale, shift [cols] or [groups, cols], a vector for each
    rows / groups rows.  pre_w None: no norm behind the sum, h is None.  y, h: tensors to fill (y may be x or branch)."""
    return _binding.residual_norm(x, branch, pre_w, post_w, gate, scale, shift, alpha, eps, y, h)


class Decoder:
    """Continues prompts through the decoder blocks, a row of every sequence at a time, over cached keys and values.

    weights: Weights (or GgufWeights).  max_seqs sequences of at most max_tokens rows each; kind: how keys and values are kept (KvCache).
    prompt() and step() return rows behind the final norm, [rows, hidden] bf16, enqueue on the library's current stream and return at once; they cannot be captured."""

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
            s = self._scratch[key] = _zeros(need, self.device)
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
            self._table[seq] = _to_gpu(pages + [0] * (self.width - len(pages)), self.device)

    def _not_captured(self, what):
        if lib.o1_capture_id():
            raise O1Error(f"Decoder.{what}: lengths and pages are the host's, which a graph would not see (capture o1_decode_step with tables on the GPU)")

    def _slots(self, seq, n):
        """Slots and numbers of a sequence's first n rows."""
        t = torch.arange(n, device=self.device)
        return self._table[seq].long()[t // self.page_size] * self.page_size + t % self.page_size, t

    def prompt(self, ids):
        """A new sequence of rows ids [n] (int64): (its name, hidden rows [n, hidden])."""
        n = ids.numel()
        if ids.dtype is not I64 or ids.dim() != 1 or n == 0 or not ids.is_cuda:
            raise O1Error("Decoder.prompt: ids int64 [n] on the GPU wanted, n > 0")
        if len(self._pages) == self.max_seqs:
            raise O1Error(f"Decoder.prompt: {self.max_seqs} sequences are open")
        self._not_captured("prompt")
        seq = self._next
        self._pages[seq], self._len[seq], self._table[seq] = [], n, None
        try:
            self._grow(seq, n)
            with _on_library(self.device):
                slots, t = self._slots(seq, n)
                pos, ids = t.float().expand(3, n).contiguous(), ids.contiguous()
                out = torch.empty(n, self.dims[2], dtype=BF16, device=self.device)
                s = self._room(n)
                check(lib.o1_prompt_rows(C.byref(self.w.binding), self._c, ptr(ids), ptr(pos), ptr(slots), ptr(s), s.numel(), ptr(out), n, *self.dims),
                      "o1_prompt_rows")
        except BaseException:        # its name would reach nobody
            self.close(seq)
            raise
        self._next += 1
        return seq, out

    def step(self, seqs, ids):
        """One new row of each sequence in seqs (all different), ids [len(seqs)] (int64): hidden rows [len(seqs), hidden]."""
        n = len(seqs)
        if ids.dtype is not I64 or ids.dim() != 1 or ids.numel() != n or not ids.is_cuda or len(set(seqs)) != n:
            raise O1Error("Decoder.step: ids int64, one for each of different sequences, on the GPU wanted")
        self._not_captured("step")
        for s in seqs:
            if s not in self._pages:
                raise O1Error(f"Decoder.step: no sequence {s}")
            self._grow(s, self._len[s] + 1)
        with _on_library(self.device):
            lens = _to_gpu([self._len[s] + 1 for s in seqs], self.device)
            pages = torch.stack([self._table[s] for s in seqs]) if n else torch.zeros(0, self.width, dtype=I32, device=self.device)
            pos, ids = (lens - 1).float().expand(3, n).contiguous(), ids.contiguous()
            out = torch.empty(n, self.dims[2], dtype=BF16, device=self.device)
            s = self._room(n)
            check(lib.o1_decode_step(C.byref(self.w.binding), self._c, ptr(ids), ptr(pos), ptr(pages), self.width, self.width, ptr(lens), ptr(s), s.numel(),
                                     ptr(out), n, *self.dims), "o1_decode_step")
        for name in seqs:            # (rows of a call that has failed are not counted: the next one writes them)
            self._len[name] += 1
        return out

    def rows(self, seq, layer):
        """(keys, values) [rows, kv_heads, 128] bf16 that a layer keeps of a sequence, as KvCache.read gives them."""
        if seq not in self._pages:
            raise O1Error(f"Decoder.rows: no sequence {seq}")
        with _on_library(self.device):
            return self.caches[layer].read(self._slots(seq, self._len[seq])[0])

    def close(self, seq):
        """Gives a sequence's pages back.  (Calls on other streams that still read them are the caller's to wait for.)"""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._len[seq], self._table[seq]
