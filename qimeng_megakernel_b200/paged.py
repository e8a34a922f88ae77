"""Paged KV cache whose sequences share a prefix: block tables, slot maps and the attention that reads it.

The pool of one layer is `[num_pages, page_size, NKV, HD]` bf16.  A sequence's block table names the page of every
`page_size` positions; sequences that start with the same tokens name the same pages for them, so a shared prompt is
stored once and `prefix_attention` reads it once for the whole batch:

    tables = build_block_tables(lengths, free_pages, page_size=64, max_pages=40, prefix_table=prefix_pages)
    step   = build_slot_map(tables.tables, kv_lengths, new_lengths, page_size=64, tokens=T)
    # K and V rows of the step's tokens go to step.slots (row page * page_size + offset of the pool) ...
    out    = prefix_attention(q, k_pages, v_pages, tables.tables, step.kv_lengths, step.cu_tokens,
                              prefix_table=prefix_pages, prefix_len=len(prefix_pages) * 64)

All three are one call into libqmk_b200.so on the current stream of the tensors' device; nothing is copied to the host,
so a step can be captured into a CUDA graph.  CUDA tensors only: there is no CPU path.  `run_prefill_synthetic(...,
shared_prefix=n)` sets up a decode state on this cache, which `decode()` then runs.

The reference keeps one contiguous cache per sequence (qimeng_megakernel/models/LLM/llama/llama3_2__1b/A100/
multi_batch/decode_schedule/globs.py:27-28); this module has no counterpart there.
"""
from __future__ import annotations

import functools
import math
import struct
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from . import _lib

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)
MAX_GROUP = 16            # query heads per KV head
MAX_HEADS = 1024          # query heads
MAX_SEQS = 1536           # requests of one attention call
MAX_TOKENS = 1 << 20      # rows of one attention call
MAX_LENGTH = 1 << 30      # positions of a sequence
# block tables and slot maps
MAX_TABLE_SEQS, MAX_TABLE_PAGES, MAX_TABLE_TOKENS = 1 << 20, 1 << 30, 1 << 24


@dataclass
class BlockTables:
    tables: torch.Tensor       # int32 [seqs, max_pages], -1 where there is no page
    used: torch.Tensor         # int32 [2]: pages taken from the free list, rows cut off at max_pages

    @classmethod
    def empty(cls, seqs: int, max_pages: int, device) -> "BlockTables":
        return cls(torch.empty(seqs, max_pages, dtype=torch.int32, device=device),
                   torch.empty(2, dtype=torch.int32, device=device))


@dataclass
class SlotMap:
    slots: torch.Tensor        # int64 [tokens]: row of the pool, -1 where there is none
    positions: torch.Tensor    # int32 [tokens]
    seq_ids: torch.Tensor      # int32 [tokens], -1 behind the last token
    active: torch.Tensor       # uint8 [tokens]: 1 where the token has a slot
    cu_tokens: torch.Tensor    # int32 [seqs + 1]: first token of every request
    kv_lengths: torch.Tensor   # int32 [seqs]: tokens in the cache after the step

    @classmethod
    def empty(cls, seqs: int, tokens: int, device) -> "SlotMap":
        i32 = lambda n: torch.empty(n, dtype=torch.int32, device=device)
        return cls(torch.empty(tokens, dtype=torch.int64, device=device), i32(tokens), i32(tokens),
                   torch.empty(tokens, dtype=torch.uint8, device=device), i32(seqs + 1), i32(seqs))


# The library's argument structures, packed in one call (the ctypes structures of _lib take several times as long to fill).
_TABLES = struct.Struct("@5P5i0P")
_SLOTS = struct.Struct("@9P4i0P")
_ATTENTION = struct.Struct("@9P2q9ifPq0P")


def _flat(n: int | None, *tensors) -> bool:
    """Contiguous int32 vectors (of n entries) all of them: the quick form of _check, which says what is wrong."""
    try:
        for t in tensors:
            if t.dtype is not torch.int32 or t.ndim != 1 or not t.is_contiguous() or (n is not None and t.shape[0] != n):
                return False
    except AttributeError:
        return False
    return True


def _check(name: str, t, dtype: torch.dtype, dim: int) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.dim() != dim:
        raise ValueError(f"{name}: expected {dim} dimensions, got shape {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _on(index: int, names: str, *tensors) -> None:
    """Every tensor of the call is on CUDA device `index` (the last check: what it says is about a call that is right otherwise)."""
    if index < 0:
        raise ValueError("the tensors must be CUDA tensors (there is no CPU path)")
    for i, t in enumerate(tensors):
        if t is not None and t.get_device() != index:
            raise ValueError(f"{names.split()[i]} is on {t.device}, expected cuda:{index}")


def _page_size(page_size: int) -> int:
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size}: expected one of {PAGE_SIZES}")
    return int(page_size)


# (the raw handle: building a torch.cuda.Stream takes longer than the rest of a call's preparation)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _call(fn, args: bytes, index: int) -> None:
    code = fn(args, index, _stream(index))
    if code != 0:
        raise _lib.QmkError(code, _lib.load().qmk_paged_last_cuda_error().decode())


def build_block_tables(lengths: torch.Tensor, free_pages: torch.Tensor, *, page_size: int, max_pages: int,
                       prefix_table: torch.Tensor | None = None, out: BlockTables | None = None) -> BlockTables:
    """Block tables for requests that need room for `lengths` tokens each (int32 [seqs], the shared prefix included).

    Row s gets min(ceil(lengths[s] / page_size), max_pages) pages: first those of `prefix_table` (int32), then pages of
    `free_pages` (int32) in order, behind those of the rows before it; the rest of the row is -1.  `used` holds the
    pages taken from `free_pages` (more than there are when it ran out: the entries it could not give are -1) and the
    number of rows cut off at `max_pages`.  No tensor of `out` may cover part of another one of the call."""
    if not _flat(None, lengths, free_pages):
        _check("lengths", lengths, torch.int32, 1)
        _check("free_pages", free_pages, torch.int32, 1)
    seqs, max_pages, shared, page_size = lengths.shape[0], int(max_pages), 0, _page_size(page_size)
    if prefix_table is not None:
        _check("prefix_table", prefix_table, torch.int32, 1)
        shared = prefix_table.shape[0]
    if seqs < 1:
        raise ValueError("lengths: no requests")
    if seqs > MAX_TABLE_SEQS:
        raise ValueError(f"lengths: {seqs} requests, expected at most {MAX_TABLE_SEQS}")
    if free_pages.shape[0] >= 1 << 31:
        raise ValueError(f"free_pages: {free_pages.shape[0]} pages, expected fewer than {1 << 31}")
    if not 1 <= max_pages <= MAX_TABLE_PAGES:
        raise ValueError(f"max_pages {max_pages}: expected 1..{MAX_TABLE_PAGES}")
    if shared > max_pages:
        raise ValueError(f"prefix_table has {shared} pages, more than max_pages = {max_pages}")
    if out is None:
        out = BlockTables.empty(seqs, max_pages, lengths.device)
    else:
        _check("out.tables", out.tables, torch.int32, 2)
        _check("out.used", out.used, torch.int32, 1)
        if out.tables.shape != (seqs, max_pages) or out.used.shape != (2,):
            raise ValueError(f"out: expected tables {(seqs, max_pages)} and used (2,), got {tuple(out.tables.shape)} "
                             f"and {tuple(out.used.shape)}")
    index = lengths.get_device()
    _on(index, "free_pages prefix_table out.tables out.used", free_pages, prefix_table, out.tables, out.used)
    args = _TABLES.pack(lengths.data_ptr(), free_pages.data_ptr(), prefix_table.data_ptr() if shared else 0,
                        out.tables.data_ptr(), out.used.data_ptr(), seqs, free_pages.shape[0], shared, page_size, max_pages)
    _call(_lib.load().qmk_build_block_tables, args, index)
    return out


def build_slot_map(block_tables: torch.Tensor, kv_lengths: torch.Tensor, new_lengths: torch.Tensor, *, page_size: int,
                   tokens: int, out: SlotMap | None = None) -> SlotMap:
    """Where the K and V rows of a step's new tokens go: request s holds `kv_lengths[s]` tokens and appends
    `new_lengths[s]` (both int32 [seqs]).  The step's tokens are numbered request by request; `tokens` is the room of the
    outputs: what does not fit is cut off (the request that straddles it appends fewer), what is left over is filled
    with slot -1, position 0, request -1, inactive.  No tensor of `out` may cover part of another one of the call."""
    _check("block_tables", block_tables, torch.int32, 2)
    seqs, max_pages = block_tables.shape
    if not _flat(seqs, kv_lengths, new_lengths):
        _check("kv_lengths", kv_lengths, torch.int32, 1)
        _check("new_lengths", new_lengths, torch.int32, 1)
    tokens, page_size = int(tokens), _page_size(page_size)
    if seqs < 1 or max_pages < 1:
        raise ValueError(f"block_tables: empty shape {tuple(block_tables.shape)}")
    if seqs > MAX_TABLE_SEQS or max_pages > MAX_TABLE_PAGES:
        raise ValueError(f"block_tables: shape {tuple(block_tables.shape)}, expected at most {MAX_TABLE_SEQS} requests with "
                         f"{MAX_TABLE_PAGES} pages")
    if kv_lengths.shape[0] != seqs or new_lengths.shape[0] != seqs:
        raise ValueError(f"kv_lengths and new_lengths: expected {seqs} requests, got {kv_lengths.shape[0]} and "
                         f"{new_lengths.shape[0]}")
    if not 1 <= tokens <= MAX_TABLE_TOKENS:
        raise ValueError(f"tokens {tokens}: expected 1..{MAX_TABLE_TOKENS}")
    if out is None:
        out = SlotMap.empty(seqs, tokens, block_tables.device)
    elif not (_flat(tokens, out.positions, out.seq_ids) and _flat(seqs, out.kv_lengths) and _flat(seqs + 1, out.cu_tokens)
              and out.slots.dtype is torch.int64 and out.slots.shape == (tokens,) and out.slots.is_contiguous()
              and out.active.dtype is torch.uint8 and out.active.shape == (tokens,) and out.active.is_contiguous()):
        for name, dtype, n in (("slots", torch.int64, tokens), ("positions", torch.int32, tokens),
                               ("seq_ids", torch.int32, tokens), ("active", torch.uint8, tokens),
                               ("cu_tokens", torch.int32, seqs + 1), ("kv_lengths", torch.int32, seqs)):
            t = getattr(out, name)
            _check(f"out.{name}", t, dtype, 1)
            if t.shape[0] != n:
                raise ValueError(f"out.{name}: expected {n} entries, got {t.shape[0]}")
    if out.kv_lengths.data_ptr() == kv_lengths.data_ptr():
        raise ValueError("out.kv_lengths must not be kv_lengths itself")
    if out.kv_lengths.data_ptr() == new_lengths.data_ptr():
        raise ValueError("out.kv_lengths must not be new_lengths itself")
    index = block_tables.get_device()
    _on(index, "kv_lengths new_lengths out.slots out.positions out.seq_ids out.active out.cu_tokens out.kv_lengths", kv_lengths,
        new_lengths, out.slots, out.positions, out.seq_ids, out.active, out.cu_tokens, out.kv_lengths)
    args = _SLOTS.pack(block_tables.data_ptr(), kv_lengths.data_ptr(), new_lengths.data_ptr(), out.slots.data_ptr(),
                       out.positions.data_ptr(), out.seq_ids.data_ptr(), out.active.data_ptr(), out.cu_tokens.data_ptr(),
                       out.kv_lengths.data_ptr(), seqs, tokens, page_size, max_pages)
    _call(_lib.load().qmk_build_slot_map, args, index)
    return out


def _rows(name: str, t) -> None:
    """[tokens, heads, head_dim] bf16 whose tokens may be any distance apart (a slice of a wider row)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name}: expected {torch.bfloat16}, got {t.dtype}")
    if t.dim() != 3:
        raise ValueError(f"{name}: expected [tokens, heads, head_dim], got shape {tuple(t.shape)}")
    tokens, heads, size = t.shape
    stride = t.stride()
    if (stride[2] != 1 or (heads > 1 and stride[1] != size) or
            (tokens > 1 and (stride[0] % 8 != 0 or stride[0] < heads * size)) or t.data_ptr() % 16 != 0):
        raise ValueError(f"{name}: heads and dimensions must be contiguous, tokens a multiple of 8 elements apart and the "
                         f"data 16-byte aligned; got strides {stride}")


@functools.lru_cache(maxsize=256)
def _workspace_bytes(tokens: int, seqs: int, heads: int, kv_heads: int, size: int, prefix_len: int, index: int) -> int:
    n = _lib.load().qmk_prefix_attention_workspace(tokens, seqs, heads, kv_heads, size, prefix_len, index)
    if n < 0:
        raise _lib.QmkError(int(n))
    return int(n)


def attention_workspace(q: torch.Tensor, k_pages: torch.Tensor, seqs: int, *, prefix_len: int = 0) -> torch.Tensor:
    """The workspace of `prefix_attention` for calls with these shapes: a program that keeps it saves the allocation.  Calls
    that may run at the same time (two streams, two captured graphs) need one each."""
    _on(q.get_device(), "k_pages", k_pages)
    n = _workspace_bytes(q.shape[0], int(seqs), q.shape[1], k_pages.shape[2], q.shape[2], int(prefix_len), q.get_device())
    return torch.empty(n, dtype=torch.uint8, device=q.device)


def prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_tables: torch.Tensor,
                     kv_lengths: torch.Tensor, cu_tokens: torch.Tensor, *, prefix_table: torch.Tensor | None = None,
                     prefix_len: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
                     lse: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a step's rows `q` [tokens, NH, HD] over the paged cache, causal inside a request.

    Request s has the rows cu_tokens[s] .. cu_tokens[s + 1] - 1 and `kv_lengths[s]` tokens in the cache, its rows'
    included; its row i sees the positions below kv_lengths[s] - rows + i + 1.  Positions below `prefix_len` (a multiple
    of the page size) are read through `prefix_table`, once for all requests; the others through `block_tables`, whose
    entries below prefix_len are not read.  A row that sees nothing gets zeros (lse: minus infinity).  Rows from
    cu_tokens[seqs] on are left as they were in `out` and `lse` (a new `out` holds zeros there).  cu_tokens must ascend from 0 to
    at most `tokens`, as build_slot_map makes it: where it does not, all rows become NaN.  `out` may be `q` itself.  A page index outside the
    pool reads as zeros.  What the last page holds behind a request's last token is never used; a non-finite V row
    inside a request may reach every row of its step.

    A NaN among a row's scores, or one of plus infinity, makes the row and its lse NaN; keys of minus infinity count as absent (a row
    that has no others sees nothing).
    At most 1024 query heads; the room of the prefix and the tables (max_pages * page size, whatever the lengths are) times the rows
    is limited by what the device counts in 32 bits: 1536 short requests of 16384 rows at 32/8 heads may have room for 880,000 positions
    each, 64 rows of 64 requests for 89 million; a call beyond that is refused.

    scale: 1 / sqrt(HD) by default.  lse: optional float32 [tokens, NH], receives the natural logarithm of the sum of
    exponentials.  Sums are held in 32 bits; probabilities are rounded to bf16 before they meet V.  Inference only."""
    _rows("q", q)
    _check("k_pages", k_pages, torch.bfloat16, 4)
    _check("v_pages", v_pages, torch.bfloat16, 4)
    _check("block_tables", block_tables, torch.int32, 2)
    if not _flat(None, kv_lengths, cu_tokens):
        _check("kv_lengths", kv_lengths, torch.int32, 1)
        _check("cu_tokens", cu_tokens, torch.int32, 1)
    tokens, heads, size = q.shape
    num_pages, page_size, kv_heads, kv_size = k_pages.shape
    seqs, max_pages = block_tables.shape
    prefix_len = int(prefix_len)
    if k_pages.shape != v_pages.shape:
        raise ValueError(f"k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)} differ")
    if size not in HEAD_DIMS or kv_size != size:
        raise ValueError(f"head_dim {size} (cache {kv_size}): expected one of {HEAD_DIMS}")
    if tokens > MAX_TOKENS:
        raise ValueError(f"{tokens} rows: expected at most {MAX_TOKENS}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads != 0 or heads // kv_heads > MAX_GROUP:
        raise ValueError(f"{heads} query heads over {kv_heads} KV heads: expected 1..{MAX_GROUP} per KV head")
    if heads > MAX_HEADS:
        raise ValueError(f"{heads} query heads: expected at most {MAX_HEADS} query heads")
    if max_pages < 1 or num_pages < 1:
        raise ValueError("block_tables and pages must not be empty")
    if not 1 <= seqs <= MAX_SEQS:
        raise ValueError(f"{seqs} requests: expected 1..{MAX_SEQS} requests")
    if kv_lengths.shape[0] != seqs or cu_tokens.shape[0] != seqs + 1:
        raise ValueError(f"expected kv_lengths [{seqs}] and cu_tokens [{seqs + 1}], got {kv_lengths.shape[0]} and "
                         f"{cu_tokens.shape[0]}")
    if not 0 <= prefix_len <= MAX_LENGTH or prefix_len % _page_size(page_size) != 0:
        raise ValueError(f"prefix_len {prefix_len}: expected whole pages of {page_size}, at most {MAX_LENGTH} positions")
    if max_pages * page_size > MAX_LENGTH:
        raise ValueError(f"block_tables: {max_pages} pages of {page_size}, expected at most {MAX_LENGTH} positions")
    if prefix_len:
        if prefix_table is None:
            raise ValueError("prefix_len needs a prefix_table")
        _check("prefix_table", prefix_table, torch.int32, 1)
        if prefix_table.shape[0] * page_size < prefix_len:
            raise ValueError(f"prefix_table has {prefix_table.shape[0]} pages, prefix_len needs {prefix_len // page_size}")
    if scale is None:
        scale = 1.0 / math.sqrt(size)
    elif not (2.0 ** -149 <= scale and scale * 1.4426950408889634 < 3.4028235e38):     # (log2(e) * scale, in 32 bits)
        raise ValueError(f"scale {scale}: expected a positive number")
    if (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad) and torch.is_grad_enabled():
        raise RuntimeError("prefix_attention has no gradient: call it under torch.inference_mode() or torch.no_grad()")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in (q, k_pages, v_pages)):
        raise RuntimeError("prefix_attention has no gradient: a tangent of its inputs would be lost")
    if out is None:
        out = torch.zeros(tokens, heads, size, dtype=torch.bfloat16, device=q.device)
    else:
        _rows("out", out)
        if out.shape != q.shape:
            raise ValueError(f"out: expected shape {tuple(q.shape)}, got {tuple(out.shape)}")
    if workspace is not None:
        _check("workspace", workspace, torch.uint8, 1)
    if lse is not None:
        _check("lse", lse, torch.float32, 2)
        if lse.shape != (tokens, heads):
            raise ValueError(f"lse: expected shape {(tokens, heads)}, got {tuple(lse.shape)}")
    index = q.get_device()
    _on(index, "k_pages v_pages block_tables kv_lengths cu_tokens prefix_table out lse workspace", k_pages, v_pages, block_tables,
        kv_lengths, cu_tokens, prefix_table if prefix_len else None, out, lse, workspace)
    if tokens == 0:
        return out
    need = _workspace_bytes(tokens, seqs, heads, kv_heads, size, prefix_len, index)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    elif workspace.shape[0] < need:
        raise ValueError(f"workspace has {workspace.shape[0]} bytes, the call needs {need}")
    one = tokens == 1                        # (the stride of a single token means nothing)
    args = _ATTENTION.pack(q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), k_pages.data_ptr(),
                           v_pages.data_ptr(), block_tables.data_ptr(), kv_lengths.data_ptr(), cu_tokens.data_ptr(),
                           prefix_table.data_ptr() if prefix_len else 0, heads * size if one else q.stride(0),
                           heads * size if one else out.stride(0), tokens, seqs, heads, kv_heads, size, page_size,
                           num_pages, max_pages, prefix_len, scale, workspace.data_ptr(), workspace.shape[0])
    _call(_lib.load().qmk_prefix_attention, args, index)
    return out


class PagedState:
    """The paged cache of a decode request: tables, lengths and the rows of the current step.

    `advance(new_lengths)` makes the slot map of a step that appends new_lengths[s] tokens to sequence s; the kernel call
    on the Globals that carry the state (`mk(globs)`) then runs that step.  All buffers of the step stay where they are from
    step to step, so the kernel's binding holds, and a graph that captured advance() and the kernel call is one more step
    every time it is replayed.  `step.kv_lengths` is what the cache holds with the last step's tokens; who writes other
    lengths there goes on from them."""

    def __init__(self, block_tables: torch.Tensor, lengths: torch.Tensor, rows: int, page_size: int,
                 prefix_table: torch.Tensor | None, prefix_len: int):
        self.block_tables, self.page_size, self.rows = block_tables, _page_size(page_size), int(rows)
        self.prefix_table, self.prefix_len = prefix_table, int(prefix_len)
        self.step: SlotMap | None = None
        self.check()
        device, seqs = block_tables.device, block_tables.shape[0]
        if not isinstance(lengths, torch.Tensor) or lengths.shape != (seqs,):
            raise ValueError(f"lengths: expected one for each of {seqs} requests")
        self.step = SlotMap.empty(seqs, self.rows, device)
        for t in (self.step.positions, self.step.active, self.step.seq_ids, self.step.cu_tokens):
            t.zero_()
        self.step.slots.fill_(-1)
        self.step.kv_lengths.copy_(lengths)
        self.ones = torch.ones(seqs, dtype=torch.int32, device=device)
        self.workspace: torch.Tensor | None = None

    def check(self) -> None:
        """Everything that the library takes as a bare address is what its kernels read.  (At construction, and again by the
        kernel call when a tensor has been put in another's place.)"""
        _check("block_tables", self.block_tables, torch.int32, 2)
        seqs, max_pages = self.block_tables.shape
        if seqs < 1 or max_pages < 1:
            raise ValueError(f"block_tables: empty shape {tuple(self.block_tables.shape)}")
        if seqs > MAX_SEQS:
            raise ValueError(f"{seqs} requests: expected 1..{MAX_SEQS} requests")
        if self.rows < 1:
            raise ValueError(f"rows {self.rows}: expected at least one")
        if not 0 <= self.prefix_len <= MAX_LENGTH or self.prefix_len % self.page_size != 0:
            raise ValueError(f"prefix_len {self.prefix_len}: expected whole pages of {self.page_size}, at most {MAX_LENGTH} positions")
        tensors = []
        if self.prefix_len:
            if self.prefix_table is None:
                raise ValueError("prefix_len needs a prefix_table")
            _check("prefix_table", self.prefix_table, torch.int32, 1)
            if self.prefix_table.shape[0] * self.page_size < self.prefix_len:
                raise ValueError(f"prefix_table has {self.prefix_table.shape[0]} pages, prefix_len needs {self.prefix_len // self.page_size}")
            tensors.append(("prefix_table", self.prefix_table))
        if self.step is not None:
            for name, dtype, n in (("slots", torch.int64, self.rows), ("positions", torch.int32, self.rows),
                                   ("seq_ids", torch.int32, self.rows), ("active", torch.uint8, self.rows),
                                   ("cu_tokens", torch.int32, seqs + 1), ("kv_lengths", torch.int32, seqs)):
                t = getattr(self.step, name)
                _check(f"step.{name}", t, dtype, 1)
                if t.shape[0] != n:
                    raise ValueError(f"step.{name}: expected {n} entries, got {t.shape[0]}")
                tensors.append((f"step.{name}", t))
        for name, t in tensors:
            if t.device != self.block_tables.device:
                raise ValueError(f"{name} is on {t.device}, expected {self.block_tables.device}")

    @property
    def capacity(self) -> int:
        """Positions a sequence's table has room for."""
        return self.block_tables.shape[1] * self.page_size

    def advance(self, new_lengths: torch.Tensor | None = None) -> SlotMap:
        """The step in which sequence s appends new_lengths[s] tokens (one each by default).  A refused call changes nothing."""
        # (a copy on the stream, in a captured graph too: the map's CTAs read the lengths while it writes the new ones)
        return build_slot_map(self.block_tables, self.step.kv_lengths.clone(), self.ones if new_lengths is None else new_lengths,
                              page_size=self.page_size, tokens=self.rows, out=self.step)

    def step_args(self, heads: int, kv_heads: int, size: int) -> _lib.PagedStepArgs:
        """The step's arguments for the library; makes the workspace on the first call."""
        device = self.block_tables.device
        if self.workspace is None:
            self.workspace = torch.empty(_workspace_bytes(self.rows, self.block_tables.shape[0], heads, kv_heads, size,
                                                          self.prefix_len, device.index), dtype=torch.uint8, device=device)
        s = self.step
        return _lib.PagedStepArgs(self.block_tables.data_ptr(), s.kv_lengths.data_ptr(), s.cu_tokens.data_ptr(),
                                  s.slots.data_ptr(), self.prefix_table.data_ptr() if self.prefix_len else None,
                                  self.block_tables.shape[0], self.block_tables.shape[1], self.prefix_len,
                                  self.workspace.data_ptr(), self.workspace.shape[0])
