"""Steps that add any number of tokens to every request: slot maps and attention over the paged int8 latent cache.

The reference's kernels add one token per request and its harness fixes the slots on the host
(kernels/layer_bench/ffn_kernel/baseline_kernel.py:38-53, kernels/layer_bench/fd_kernel/flash_decoding.py:3-57).  Here a
request gets one or many tokens per step -- a prompt, a piece of one, drafted tokens to verify -- with the same field names:

  * ``chunk_maps`` finds the slots of the new tokens from the request lengths, on the device;
  * ``cache_append`` (attention.py) writes their latents there;
  * ``chunk_attention_int8_latent_absorb`` lets them attend to everything cached before them and to one another,
    with a causal, window, prefix or document mask, capped scores and a bias by distance.

Argument checking and pointer plumbing only; the arithmetic runs in the CUDA kernels of ``liblsvd_b200.so``.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from .attention import InferState, LatentCacheLayout, _require_cuda, _stream_ptr


class ChunkMaps(NamedTuple):
    """What a step's tokens need (see ``chunk_maps``)."""
    b_start_loc: torch.Tensor        # [B + 1] first token row of every request; the last entry is the number of tokens
    b_seq_len: torch.Tensor          # [B] lengths with the new tokens
    mem_index: torch.Tensor          # [num_tokens] cache slot of every token, -1 behind the last one
    position_ids: torch.Tensor       # [num_tokens] position of every token in its request, 0 behind the last one
    free_head: Optional[torch.Tensor]    # [1] entries of free_pages taken, or None without a free list


def _i32(name, t, *shape, device):
    if t.dtype != torch.int32 or not t.is_contiguous() or (shape and tuple(t.shape) != shape):
        raise ValueError(f"{name} must be a contiguous int32 tensor" + (f" of shape {list(shape)}" if shape else ""))
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    return t.data_ptr()


def _bound(n) -> int:
    """A bound as the C side holds it: one beyond 32 bits bounds nothing, and must not come out as its lower half."""
    return min(int(n), 2 ** 31 - 1)


def _status(t, device):
    """Address of a status word: the kernels write to it, so it has to be where they run."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.numel() < 1 or t.device != device:
        raise ValueError(f"status_word must be an int32 tensor on {device}")
    return t.data_ptr()


def _table(name, t, device):
    if t.dtype != torch.int32 or t.dim() != 2 or t.stride(1) != 1 or t.device != device or t.numel() == 0:
        raise ValueError(f"{name} must be a non-empty int32 table [rows, columns] with unit column stride on {device}")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"rows of {name} must not overlap")
    return t.data_ptr(), t.stride(0)


@torch.no_grad()
def chunk_maps(b_req_idx, b_ready_cache_len, b_new_len, block_table, page_size: int, req_to_token, num_tokens: int, num_slots: int,
               free_pages=None, free_head=None, rebuild: bool = False, out: Optional[ChunkMaps] = None,
               alloc_tensor_func=torch.empty, status_word=None, max_new_in_batch: int = 0) -> ChunkMaps:
    """Slots and positions of the tokens that a step adds, from the request lengths, in one launch.

    Entry b of the batch is row ``b_req_idx[b]`` of the tables, holds ``b_ready_cache_len[b]`` tokens and gets
    ``b_new_len[b]`` more.  Pages of ``page_size`` slots that it needs beyond the ones it has come from
    ``free_pages[free_head:]`` in batch order and are entered into ``block_table [rows, max_blocks]`` (without a free list,
    ``free_pages`` None, the table lists every page already; a free list of no entries has run out); ``req_to_token [rows, width]`` gets the slots of the new positions -- of all positions
    with ``rebuild``, for pages that were taken over from elsewhere.  All tensors are int32 on one device; ``num_tokens`` is
    the capacity of the token maps and ``num_slots`` the number of cache rows.  ``out`` receives the results;
    ``out.b_seq_len`` may be ``b_ready_cache_len`` and ``out.free_head`` may be ``free_head``, so that a captured step
    advances the lengths at every replay.  An entry that does not fit (its row, its length, ``num_tokens``, more new tokens
    than a ``max_new_in_batch`` above zero, the free pages, a row that an earlier entry adds tokens to, or, in
    a rebuild, no new tokens and more cached ones than the entry that adds tokens to its row) gets no page and slot -1 for its tokens, its length stays, and
    ``LSVD_ERR_BOUNDS`` is written to ``status_word``.
    """
    _require_cuda(b_req_idx, b_ready_cache_len, b_new_len, block_table, req_to_token, free_pages, free_head)
    dev, B = b_req_idx.device, b_req_idx.numel()
    if (free_pages is None) != (free_head is None):
        raise ValueError("free_pages and free_head go together")
    if B == 0 or num_tokens < 0 or max_new_in_batch < 0:
        raise ValueError("an empty batch or a negative number of tokens")
    if block_table.shape[0] != req_to_token.shape[0]:
        raise ValueError("block_table and req_to_token must have the same number of rows")
    if out is None:
        new = lambda n: alloc_tensor_func((n,), dtype=torch.int32, device=dev)
        out = ChunkMaps(new(B + 1), new(B), new(num_tokens), new(num_tokens), new(1) if free_pages is not None else None)
    a = _lib.ChunkMapsArgs()
    a.batch, a.page_size, a.num_tokens, a.num_slots = B, page_size, num_tokens, num_slots
    a.b_req_idx = _i32("b_req_idx", b_req_idx, B, device=dev)
    a.b_ready_cache_len = _i32("b_ready_cache_len", b_ready_cache_len, B, device=dev)
    a.b_new_len = _i32("b_new_len", b_new_len, B, device=dev)
    a.block_table, a.block_table_stride = _table("block_table", block_table, dev)
    a.req_to_token, a.req_to_token_stride = _table("req_to_token", req_to_token, dev)
    a.max_blocks, a.table_rows, a.max_len = block_table.shape[1], block_table.shape[0], req_to_token.shape[1]
    a.rebuild, a.max_new_in_batch = int(rebuild), _bound(max_new_in_batch)
    if free_pages is not None:
        a.free_pages, a.num_free = _i32("free_pages", free_pages, free_pages.numel(), device=dev), free_pages.numel()
        a.free_head = _i32("free_head", free_head, 1, device=dev)
        if out.free_head is None:
            raise ValueError("out.free_head is needed with a free list")
        a.free_head_out = _i32("out.free_head", out.free_head, 1, device=dev)
    a.b_start_loc = _i32("out.b_start_loc", out.b_start_loc, B + 1, device=dev)
    a.b_seq_len = _i32("out.b_seq_len", out.b_seq_len, B, device=dev)
    a.mem_index = _i32("out.mem_index", out.mem_index, num_tokens, device=dev)
    a.position_ids = _i32("out.position_ids", out.position_ids, num_tokens, device=dev)
    a.status_word = _status(status_word, dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().lsvd_chunk_maps(C.byref(a), _stream_ptr(b_req_idx)))
    return out


class ChunkState:
    """Batch bookkeeping of a step with several new tokens per request, with ``InferState``'s field names.

    Request b is row ``b_req_idx[b]`` of ``req_manager.req_to_token_indexs``, is ``b_seq_len[b]`` tokens long with the new
    ones, and its new tokens are the rows ``b_start_loc[b] .. b_start_loc[b + 1]`` of the step's tensors; they go to the cache
    slots ``mem_index``.  ``max_len_in_batch`` and ``max_new_in_batch`` are bounds known to the host (they size the grids).
    ``status_word`` receives what ``begin`` and the attention report (a request that was refused or skipped) unless they are given
    another one; ``check`` raises it.
    """

    def __init__(self, b_req_idx, b_seq_len, b_start_loc, req_to_token, max_len_in_batch: int, max_new_in_batch: int,
                 mem_index=None, position_ids=None):
        self.batch_size = b_req_idx.numel()
        self.max_len_in_batch, self.max_new_in_batch = int(max_len_in_batch), int(max_new_in_batch)
        self.b_req_idx, self.b_seq_len, self.b_start_loc = b_req_idx, b_seq_len, b_start_loc
        self.req_manager = InferState._ReqManager(req_to_token)
        self.mem_index, self.position_ids = mem_index, position_ids
        self.status_word = torch.zeros(1, dtype=torch.int32, device=b_req_idx.device)
        self.pages = None

    @classmethod
    def paged(cls, rows: int, max_len_in_batch: int, max_tokens: int, max_new_in_batch: int, num_pages: int, page_size: int,
              b_req_idx=None, device="cuda"):
        """An empty paged state: ``rows`` requests of up to ``max_len_in_batch`` tokens, ``num_pages`` free pages of
        ``page_size`` slots, steps of up to ``max_tokens`` tokens, ``max_new_in_batch`` of them for one request.  ``begin`` starts
        a step."""
        i32 = dict(dtype=torch.int32, device=device)
        req = torch.arange(rows, **i32) if b_req_idx is None else b_req_idx.to(**i32).contiguous()
        blocks = -(-max_len_in_batch // page_size)
        s = cls(req, torch.zeros(req.numel(), **i32), torch.zeros(req.numel() + 1, **i32),
                torch.full((rows, max_len_in_batch), -1, **i32), max_len_in_batch, max_new_in_batch,
                torch.full((max_tokens,), -1, **i32), torch.zeros(max_tokens, **i32))
        s.pages = dict(block_table=torch.full((rows, blocks), -1, **i32), page_size=page_size, num_slots=num_pages * page_size,
                       free_pages=torch.arange(num_pages, **i32), free_head=torch.zeros(1, **i32))
        return s

    def begin(self, b_new_len, rebuild: bool = False, status_word=None) -> "ChunkState":
        """Start a step that adds ``b_new_len[b]`` tokens to request b: takes pages, advances ``b_seq_len`` in place and fills
        ``b_start_loc``, ``mem_index``, ``position_ids`` and the new slots of ``req_to_token``.  One launch, no host work that
        depends on the lengths: it can be captured with the step that follows it."""
        if self.pages is None:
            raise ValueError("begin() needs a paged state (ChunkState.paged)")
        g = self.pages
        chunk_maps(self.b_req_idx, self.b_seq_len, b_new_len, g["block_table"], g["page_size"], self.req_manager.req_to_token_indexs,
                   self.mem_index.numel(), g["num_slots"], g["free_pages"], g["free_head"], rebuild,
                   ChunkMaps(self.b_start_loc, self.b_seq_len, self.mem_index, self.position_ids, g["free_head"]),
                   status_word=self.status_word if status_word is None else status_word, max_new_in_batch=self.max_new_in_batch)
        return self

    def check(self) -> None:
        """Raises ``LsvdError`` if a step since the last call has refused or skipped a request (its tokens have no slots, its rows
        no result), and forgets it.  Reads the status word on the current stream and waits for it."""
        code = int(self.status_word.item())
        if code != _lib.OK:
            self.status_word.zero_()
            _lib.check(code)


def attn_chunk_workspace_bytes(state, layout: LatentCacheLayout, num_tokens: int) -> int:
    return int(_lib.load().lsvd_attn_chunk_workspace_bytes(state.batch_size, layout.num_heads, layout.sum_v, num_tokens,
                                                           _bound(state.max_new_in_batch), _bound(state.max_len_in_batch)))


def kept_workspace(kept: list, state, layout: LatentCacheLayout, num_tokens: int, device) -> torch.Tensor:
    """The workspace for a step out of ``kept``, which grows as steps need it.  An outgrown workspace stays there: a captured step
    may still point to it (each is at least twice the last, so all of them together are at most twice the largest).
    Steps that take their workspace from one list run one after another, captured or not; for steps side by side on two streams
    give each its own ``workspace``."""
    with torch.cuda.device(device):
        need = max(attn_chunk_workspace_bytes(state, layout, num_tokens), 256)
    here = [w for w in kept if w.device == device]
    last = here[-1].numel() if here else 0
    if last < need:
        here.append(torch.empty(max(need, 2 * last), dtype=torch.uint8, device=device))
        kept.append(here[-1])
    return here[-1]


def _row_view(name, t, rows, cols, dev):
    if t.dtype != torch.float16 or tuple(t.shape) != (rows, cols) or t.stride(-1) != 1 or t.device != dev:
        raise ValueError(f"{name} must be fp16 [{rows}, {cols}] with unit inner stride on {dev}")
    return t.data_ptr(), t.stride(0)


@torch.no_grad()
def chunk_attention_int8_latent_absorb(
        q, state, q_head_num: int, head_dim: int,
        cache_latent_k, cache_latent_k_scale, cache_latent_v, cache_latent_v_scale,
        up_k, up_v=None, layout: Optional[LatentCacheLayout] = None,
        out=None, out_latent=None, alloc_tensor_func=torch.empty, workspace=None, sm_scale: Optional[float] = None,
        causal: bool = True, window: int = 0, b_prefix_len=None, key_begin=None, softcap: float = 0.0, alibi_slopes=None,
        status_word=None):
    """Attention of a step's new tokens over the int8 latent cache, any number of them per request.

    The several-token form of ``token_decode_attention_int8_latent_absorb``: same cache layouts, up-factors, outputs and
    conventions, with ``q [num_tokens, H, D]`` (or ``[num_tokens, H * D]``) holding the new tokens of all requests one after
    the other (``state.b_start_loc``).  The tokens' own latents must be in the cache.  A token at position ``pos`` sees the
    keys ``t <= pos`` of its request, and

      * ``window > 0``: only ``t > pos - window``;
      * ``b_prefix_len [B]`` int32: also every ``t`` below it (a prefix whose tokens see one another; all of them have to be
        added in one step, since an earlier piece cannot see what is not cached yet);
      * ``key_begin [num_tokens]`` int32: only ``t >= key_begin`` (first position of the token's document);
      * ``causal=False``: every key of the request (with a window: ``|pos - t| < window``).

    ``softcap > 0`` replaces a score x by ``softcap * tanh(x / softcap)``; ``alibi_slopes [H]`` fp32 subtracts
    ``slope * |pos - t|`` after that.  A token without a cache slot (``state.mem_index`` negative: ``chunk_maps`` has refused its
    request) sees nothing.  A request whose rows are not all in ``q``
    (``state.b_start_loc``) is skipped and reported.  Returns ``out [num_tokens, H, D]`` fp16 when ``up_v`` is given, otherwise the latent
    result ``[num_tokens, sum r_v]``.  Rows of tokens that see nothing are zero; rows behind the last token are not written.
    """
    _require_cuda(q, cache_latent_k, cache_latent_v, up_k, up_v, alibi_slopes, b_prefix_len, key_begin)
    dev, B = q.device, state.batch_size
    if q.dtype != torch.float16 or up_k.dtype != torch.float16 or (up_v is not None and up_v.dtype != torch.float16):
        raise ValueError("q and up-factors must be fp16")
    if q.dim() == 2 and q.shape[1] == q_head_num * head_dim:
        q = q.unflatten(1, (q_head_num, head_dim))
    if q.dim() != 3 or tuple(q.shape[1:]) != (q_head_num, head_dim):
        raise ValueError(f"q must be [num_tokens, {q_head_num}, {head_dim}], got {tuple(q.shape)}")
    if q.stride(2) != 1:
        q = q.contiguous()
    T = q.shape[0]
    if cache_latent_k.dim() == 3:
        if layout is None:
            layout = LatentCacheLayout.uniform(q_head_num, cache_latent_k.shape[-1], cache_latent_v.shape[-1])
        if not cache_latent_k.is_contiguous() or not cache_latent_v.is_contiguous():
            raise ValueError("3-D latent caches must be contiguous")
        cache_latent_k = cache_latent_k.view(cache_latent_k.shape[0], -1)
        cache_latent_v = cache_latent_v.view(cache_latent_v.shape[0], -1)
    if layout is None:
        raise ValueError("a LatentCacheLayout is needed for 2-D (ragged) caches")
    if layout.num_heads != q_head_num:
        raise ValueError("only num_q_heads == num_kv_heads is supported")
    if layout.sum_k != up_k.shape[0] or up_k.shape[1:] != (head_dim,) or (up_v is not None and up_v.shape != (layout.sum_v, head_dim)):
        raise ValueError("up-factors must be [sum r, head_dim]")
    if up_k.stride(1) != 1 or (up_v is not None and up_v.stride(1) != 1):
        raise ValueError("up-factors must have unit inner stride")
    if up_k.device != dev or (up_v is not None and up_v.device != dev):
        raise ValueError(f"up-factors must be on {dev}")
    hm, n_slots = layout.head_major, layout.num_slots_of(cache_latent_k, "k")
    for which, cache, scale, total in (("k", cache_latent_k, cache_latent_k_scale, layout.sum_k),
                                       ("v", cache_latent_v, cache_latent_v_scale, layout.sum_v)):
        if cache.dtype != torch.int8 or scale.dtype != torch.float16 or cache.device != dev or scale.device != dev:
            raise ValueError(f"cache_latent_{which} must be int8 and its scale fp16, on {dev}")
        if hm:
            if cache.numel() != n_slots * total or tuple(scale.shape) != (layout.num_heads, n_slots):
                raise ValueError("caches / scales do not match the head-major layout")
            if not cache.is_contiguous() or not scale.is_contiguous():
                raise ValueError("head-major caches and scales must be contiguous")
        else:
            if tuple(cache.shape) != (n_slots, total) or tuple(scale.shape) != (n_slots, layout.num_heads):
                raise ValueError("cache row width does not match the layout")
            if cache.stride(1) != 1 or scale.stride(1) != 1:
                raise ValueError("caches and scales must have unit inner stride")
    r2t = state.req_manager.req_to_token_indexs
    a = _lib.AttnChunkArgs()
    a.batch, a.num_heads, a.head_dim, a.num_tokens = B, q_head_num, head_dim, T
    a.max_len_in_batch, a.max_new_in_batch = _bound(state.max_len_in_batch), _bound(state.max_new_in_batch)
    a.sm_scale = float(sm_scale) if sm_scale is not None else 0.0
    a.num_slots, a.cache_layout = n_slots, _lib.CACHE_HEAD_MAJOR if hm else _lib.CACHE_SLOT_MAJOR
    a.req_to_token, a.req_to_token_stride = _table("req_to_token", r2t, dev)
    if r2t.shape[1] < a.max_len_in_batch:
        raise ValueError(f"req_to_token has {r2t.shape[1]} columns for requests of up to {a.max_len_in_batch} tokens")
    a.req_to_token_rows = r2t.shape[0]
    a.b_req_idx = _i32("b_req_idx", state.b_req_idx, B, device=dev)
    a.b_seq_len = _i32("b_seq_len", state.b_seq_len, B, device=dev)
    a.b_start_loc = _i32("b_start_loc", state.b_start_loc, B + 1, device=dev)
    if out is None and up_v is not None:
        out = alloc_tensor_func((T, q_head_num, head_dim), dtype=torch.float16, device=dev)
    if out_latent is None and up_v is None:
        out_latent = alloc_tensor_func((T, layout.sum_v), dtype=torch.float16, device=dev)
    if out is not None:
        if up_v is None:
            raise ValueError("out needs up_v; without it the result is out_latent")
        if out.dtype != torch.float16 or tuple(out.shape) != (T, q_head_num, head_dim) or out.stride(2) != 1 or out.device != dev:
            raise ValueError(f"out must be fp16 [{T}, {q_head_num}, {head_dim}] with unit inner stride on {dev}")
        a.out, a.out_stride_t, a.out_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
    if out_latent is not None:
        a.out_latent, a.out_latent_stride_t = _row_view("out_latent", out_latent, T, layout.sum_v, dev)
    a.q, a.q_stride_t, a.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    a.k_off, a.v_off = layout.off_c("k"), layout.off_c("v")
    a.cache_k, a.cache_k_row_stride = cache_latent_k.data_ptr(), 0 if hm else cache_latent_k.stride(0)
    a.scale_k, a.scale_k_row_stride = cache_latent_k_scale.data_ptr(), 0 if hm else cache_latent_k_scale.stride(0)
    a.cache_v, a.cache_v_row_stride = cache_latent_v.data_ptr(), 0 if hm else cache_latent_v.stride(0)
    a.scale_v, a.scale_v_row_stride = cache_latent_v_scale.data_ptr(), 0 if hm else cache_latent_v_scale.stride(0)
    a.up_k, a.up_k_row_stride = up_k.data_ptr(), up_k.stride(0)
    if up_v is not None:
        a.up_v, a.up_v_row_stride = up_v.data_ptr(), up_v.stride(0)
    a.causal, a.window, a.softcap = int(bool(causal)), _bound(window), float(softcap)
    if window < 0 or softcap < 0:
        raise ValueError("window and softcap must not be negative")
    if alibi_slopes is not None:
        if alibi_slopes.dtype != torch.float32 or tuple(alibi_slopes.shape) != (q_head_num,) or not alibi_slopes.is_contiguous() \
                or alibi_slopes.device != dev:
            raise ValueError(f"alibi_slopes must be a contiguous fp32 tensor [{q_head_num}] on {dev}")
        a.alibi_slopes = alibi_slopes.data_ptr()
    if b_prefix_len is not None:
        a.b_prefix_len = _i32("b_prefix_len", b_prefix_len, B, device=dev)
    slots = getattr(state, "mem_index", None)
    if slots is not None:
        if slots.numel() < T:
            raise ValueError(f"state.mem_index has {slots.numel()} slots for {T} rows")
        a.mem_index = _i32("state.mem_index", slots, device=dev)
    if key_begin is not None:
        a.key_begin = _i32("key_begin", key_begin, T, device=dev)
    with torch.cuda.device(dev):       # the workspace is sized, and the kernels run, on the tensors' device
        need = attn_chunk_workspace_bytes(state, layout, T)
        if workspace is None:
            workspace = alloc_tensor_func((max(need, 256),), dtype=torch.uint8, device=dev)
        if workspace.device != dev or not workspace.is_contiguous():
            raise ValueError(f"workspace must be a contiguous tensor on {dev}")
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        if status_word is None:
            status_word = getattr(state, "status_word", None)
        a.status_word = _status(status_word, dev)
        _lib.check(_lib.load().lsvd_attn_chunk(C.byref(a), _stream_ptr(q)))
    return out if out is not None else out_latent
