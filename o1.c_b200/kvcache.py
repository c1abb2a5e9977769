"""Rows after a prompt: a paged cache of keys and values, the attention of new rows over it, pages handed out on the GPU, rotary positions, the residual
add between two norms -- o1_kv_write, o1_kv_read, o1_kv_attention, o1_kv_pages_grow, o1_kv_pages_shrink, o1_rotary and o1_residual_norm on torch tensors -- and a
Decoder that continues prompts with them.

Like every entry point they enqueue on the library's current stream (use_torch_stream()) and return at once.  Arguments that
do not fit raise O1Error; a slot, page, sequence or length that does not fit is found on the device (lib.o1_device_error() gives 70, 71 or, with no pages left, 73).
Where torch's current stream is another one, what these calls make (caches, results, tables) is made, filled and freed in the order of the library's;
ordering that, and their inputs, with torch's own work is the caller's.
"""
import ctypes as C
import math
import os
from collections import namedtuple

import torch

_BINDING = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_binding.so")
if not os.path.exists(_BINDING):
    raise ImportError(f"{_BINDING} is missing: build it with `python o1.c_b200/build.py`. There is no fallback path.")

from . import _binding  # noqa: E402

if _binding.torch_version != torch.__version__.split("+")[0]:
    raise ImportError(f"{_BINDING} is of torch {_binding.torch_version}, this is {torch.__version__}: build it with `python o1.c_b200/build.py`")

from . import HEAD_DIM, KV_HEADS, ROPE_THETA, KvCacheC, KvPagesC, O1Error, RopeC, RopeScalingC, _on_library, check, lib, ptr  # noqa: E402

KINDS = {"bf16": (0, torch.bfloat16), "fp8": (1, torch.float8_e4m3fn), "int8": (2, torch.int8), "uint4": (4, torch.uint8)}
_BY_DTYPE = {d: n for n, d in KINDS.values()}
COUNTERS = 32768         # O1_KV_ATTENTION_COUNTERS: the bytes of a workspace that begin as zeros
BF16, I32, I64, F32 = torch.bfloat16, torch.int32, torch.int64, torch.float32
_stream = lib.o1_get_stream
Grown = namedtuple("Grown", "slots positions starts lens pages")
Grown.__doc__ = """What KvPages.grow gives: slots [rows] int64 and positions [rows] int32 of the new rows, starts [requests + 1] (where each request's rows begin), lens [requests]
and pages [requests, width] as KvCache.attend takes them.  (One allocation, which lives as long as any of them.)"""
_binding.setup(*(C.cast(f, C.c_void_p).value for f in (lib.o1_kv_write, lib.o1_kv_read, lib.o1_kv_attention, lib.o1_residual_norm, lib.o1_get_stream, lib.o1_capture_id,
                                                       lib.o1_kv_pages_grow, lib.o1_kv_pages_shrink, lib.o1_rotary)), O1Error, check, Grown)


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
        with _on_library(device):
            self.scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
            self.scratch[:COUNTERS].zero_()
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

    kind: "bf16", or "fp8" / "int8" (a byte a value and one fp32 scale for each token and head), or "uint4" (two values to a byte, uint8 [pages, kv_heads, page_size,
    64] with the first value in the low bits, and a bf16 pair (scale, least value) [pages, kv_heads, page_size, 2] for each token and head).  A token's slot is
    page * page_size + its place in the page; which pages a sequence has is the caller's table (KvPages hands them out on the GPU)."""

    def __init__(self, pages, page_size=64, kind="bf16", kv_heads=KV_HEADS, device="cuda"):
        _need(kind in KINDS, f"KvCache: kind {kind!r} (one of {', '.join(KINDS)})")
        shape = (pages, kv_heads, page_size, HEAD_DIM // 2 if kind == "uint4" else HEAD_DIM)
        dtype = KINDS[kind][1]
        with _on_library(device):
            k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) if kind != "bf16" else
                    torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
            ks, vs = (None if kind == "bf16" else torch.zeros(shape[:3] + (2,), dtype=BF16, device=device) if kind == "uint4" else
                      torch.zeros(shape[:3], device=device) for _ in range(2))
        self._set(k, v, ks, vs)

    @classmethod
    def over(cls, k, v, k_scale=None, v_scale=None):
        """A cache in tensors that the caller has."""
        self = cls.__new__(cls)
        self._set(k, v, k_scale, v_scale)
        return self

    def _set(self, k, v, k_scale, v_scale):
        _need(k.dtype in _BY_DTYPE and k.dim() == 4 and k.size(3) == (HEAD_DIM // 2 if k.dtype is torch.uint8 else HEAD_DIM),
              "KvCache: k [pages, kv_heads, page_size, 128] bf16, float8_e4m3fn or int8, or [pages, kv_heads, page_size, 64] uint8 wanted")
        _need(v.dtype == k.dtype and v.shape == k.shape, "KvCache: v differs from k in shape or type")
        kind = _BY_DTYPE[k.dtype]
        tensors = [k, v]
        if kind:
            for s in (k_scale, v_scale):
                if k.dtype is torch.uint8:
                    _need(s is not None and s.dtype is BF16 and s.shape == (*k.shape[:3], 2), "KvCache: scales [pages, kv_heads, page_size, 2] bf16 (scale, least value) wanted")
                else:
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
        need = lib.o1_kv_attention_workspace_bytes_of(self.c.type, heads, self.kv_heads)
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


class KvPages:
    """Which pages of a cache sequences have, handed out on the GPU: table [max_seqs, width] (a sequence's pages in order, -1 behind them), lens [max_seqs] (its rows),
    free [pages] (a stack of free pages) and state [2] (how many are free; the calls' own), all int32.

    Calls on the same pages follow one another.  They can be captured: a graph serves the counts and sequences that its tensors hold at each replay."""

    def __init__(self, pages, page_size=64, max_seqs=64, width=64, device="cuda"):
        _need(min(pages, max_seqs, width) > 0, "KvPages: pages, max_seqs and width must be positive")
        with _on_library(device):
            table, lens, free, state = (torch.empty(s, dtype=I32, device=device) for s in ((max_seqs, width), (max_seqs,), (pages,), (2,)))
        self._set(table, lens, free, state, page_size)
        self.reset()

    @classmethod
    def over(cls, table, lens, free, state, page_size):
        """Pages in tensors that the caller has, as they stand."""
        self = cls.__new__(cls)
        self._set(table, lens, free, state, page_size)
        return self

    def _set(self, table, lens, free, state, page_size):
        for name, t, dim in (("table", table, 2), ("lens", lens, 1), ("free", free, 1), ("state", state, 1)):
            _need(t.dtype is I32 and t.dim() == dim and t.is_cuda and t.device == table.device and t.is_contiguous() and 0 < t.numel() and max(t.shape) < 2 ** 31,
                  f"KvPages: {name} int32, of {dim} dimensions, contiguous, on one GPU wanted")
        _need(lens.size(0) == table.size(0) <= 8192 and state.size(0) == 2, "KvPages: lens [max_seqs], at most 8192, and state [2] wanted")
        _need(0 < page_size < 2 ** 31 and page_size % 16 == 0 and table.size(1) * page_size <= 2 ** 30 >= free.numel(),
              "KvPages: page_size must be a multiple of 16, and a table's rows and the pages at most 2^30")
        self.table, self.lens, self.free, self.state, self.page_size = table, lens, free, state, page_size
        self.pages, self.max_seqs, self.width = free.size(0), *table.shape
        self.device = table.device
        self.c = KvPagesC(*(t.data_ptr() for t in (table, lens, free, state)), self.pages, page_size, self.max_seqs, self.width)
        self._at, self._gpu = C.addressof(self.c), table.get_device()

    def reset(self):
        """Every page free, every sequence empty."""
        _need(torch.cuda.current_device() == self._gpu, "KvPages.reset: its memory is on another GPU than the current one")
        check(lib.o1_kv_pages_reset(C.byref(self.c)), "o1_kv_pages_reset")

    def grow(self, counts, rows, seqs=None):
        """counts [requests] int32 new rows of sequences seqs [requests] int32 (all different; None: 0, 1, ...), with room for `rows` of them in all: Grown.

        The requests' rows lie behind one another; rows behind the last one have slot -1.  A request that cannot be served (70: no such sequence, or named twice; 71: too many
        rows; 73: no pages left) has slots of -1 and a length of 0.  pages is the table itself where seqs is None."""
        return _binding.pages_grow(self._at, self._gpu, self.table, counts, rows, seqs)

    def shrink(self, keep, seqs=None):
        """Sequences seqs [requests] int32 (None: 0, 1, ...) keep their first keep [requests] int32 rows; the pages behind them are free again."""
        _binding.pages_shrink(self._at, self._gpu, keep, seqs)


class _Turned(torch.autograd.Function):
    """Rotary's call on rows that need a gradient, which is the results' turned back."""

    @staticmethod
    def forward(ctx, rope, positions, inverse, *x):
        ctx.rope, ctx.inverse = rope, inverse
        ctx.save_for_backward(positions)
        return rope(x if len(x) > 1 else x[0], positions, inverse)

    @staticmethod
    def backward(ctx, *grads):
        positions, = ctx.saved_tensors
        wanted = [i for i, needed in enumerate(ctx.needs_input_grad[3:]) if needed]
        rows = tuple(grads[i].contiguous() for i in wanted)
        # on the stream that autograd has for it, where the gradients are made
        stream = _stream()
        lib.o1_set_stream(C.c_void_p(torch.cuda.current_stream(positions.device).cuda_stream))
        try:
            turned = ctx.rope(rows if len(rows) > 1 else rows[0], positions, not ctx.inverse)
        finally:
            lib.o1_set_stream(C.c_void_p(stream))
        back = dict(zip(wanted, turned if len(rows) > 1 else (turned,)))
        return (None, None, None, *(back.get(i) for i in range(len(grads))))


class Rotary:
    """Rotary positions: the first rot_dim values of each head turned in pairs, "half" (i, i + rot_dim / 2) or "interleaved" (2i, 2i + 1), by position *
    theta^(-2i / rot_dim).  Angles are exact to position * 2^-65 turns (64-bit fractions of a turn), then rounded to fp32 once reduced.

    scaling, for contexts longer than the model was made for: {"kind": "linear", "factor": f}, {"kind": "ntk", "factor": f}, {"kind": "yarn", "factor": f, "original":
    rows, "fast": 32, "slow": 1}, or {"kind": "factors", "factors": [rot_dim / 2 divisors]}; with "attention": what results are multiplied by."""

    def __init__(self, head_dim=HEAD_DIM, rot_dim=None, theta=ROPE_THETA, layout="half", scaling=None, device="cuda"):
        rot_dim = head_dim if rot_dim is None else rot_dim
        _need(0 < rot_dim <= head_dim <= 4096 and rot_dim % 2 == 0, f"Rotary: rot_dim {rot_dim} (even, at most head_dim {head_dim}, which is at most 4096)")
        _need(layout in ("half", "interleaved"), f"Rotary: layout {layout!r} (half or interleaved)")
        scaling = dict(scaling or {"kind": "none"})
        kinds = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "factors": 4}
        kind = scaling.pop("kind", None)
        _need(kind in kinds, f"Rotary: scaling of kind {kind!r} (one of {', '.join(kinds)})")
        unknown = set(scaling) - {"factor", "original", "fast", "slow", "attention", "factors"}
        _need(not unknown, f"Rotary: scaling has no {', '.join(sorted(unknown))}")
        _need(kind in ("none", "factors") or "factor" in scaling, f"Rotary: scaling of kind {kind} has a factor")
        _need("attention" not in scaling or 0.0 < scaling["attention"] < math.inf, "Rotary: attention, what results are multiplied by, is positive and finite")
        factors = [float(f) for f in scaling.get("factors", ())]
        _need(len(factors) == (rot_dim // 2 if kind == "factors" else 0), "Rotary: factors, one for each pair, belong to scaling of that kind")
        c = RopeScalingC(kinds[kind], scaling.get("factor", 1.0), scaling.get("original", 0.0), scaling.get("fast", 32.0), scaling.get("slow", 1.0), scaling.get("attention", 0.0),
                         (C.c_double * len(factors))(*factors) if factors else None)
        turns, factor = (C.c_uint64 * (rot_dim // 2))(), C.c_float()
        check(lib.o1_rope_turns(theta, rot_dim, C.byref(c), turns, C.byref(factor)), "o1_rope_turns")
        with _on_library(device):
            self.turns = torch.frombuffer(turns, dtype=I64).to(device)
        self.factor, self.head_dim, self.rot_dim, self.layout = factor.value, head_dim, rot_dim, layout
        self.c = RopeC(self.turns.data_ptr(), factor, head_dim, rot_dim, 0 if layout == "half" else 1)
        self._at, self._gpu = C.addressof(self.c), self.turns.get_device()

    def __call__(self, x, positions, inverse=False, out=None):
        """Rows x [rows, heads, head_dim] bf16 or fp32 (rows of any pitch), or a pair of them (queries and keys), turned by positions [rows] int32 or int64.

        inverse: turned back.  out: what to fill, like x (x itself: in place; no other memory of x's, nor one another's).  (A pair's results share an allocation.)
        Rows that need a gradient get results with one (not into out)."""
        y = _binding.rotary(self._at, self._gpu, positions, inverse, x, out)
        return _Turned.apply(self, positions, bool(inverse), *(x if isinstance(x, tuple) else (x,))) if y is NotImplemented else y


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
        need = lib.o1_decode_scratch_bytes_of(self._c[0].type, rows, *self.dims[:5])
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
