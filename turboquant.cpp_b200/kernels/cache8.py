"""A key/value cache in 8 bits whose length can be bounded (csrc/cache8.cu, csrc/attention8.cu, csrc/prompt8.cu, csrc/evict.cu).

An element is an e4m3 code times 2^(b - 127), b one byte for 16 consecutive rows of a (page, plane, key/value head): the smallest power of
two, of those from 2^-126 on, under which the largest finite magnitude of the 16 rows is at most 448.  A block that takes rows in
several steps keeps the largest byte; the rows it held are then rounded again.  What is not finite becomes NaN and does not count for the byte.

    codes    [pages, 2 (keys, values), kv heads, page_size, head size] float8_e4m3fn
    scales   [pages, 2, kv heads, page_size / 16] uint8
    weights  [pages, kv heads, page_size] float32: the attention weight each row has received, where it is kept

The step's rows are packed, sequence after sequence: rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1 belong to sequence s, and row t lies at
place held[s] + t - cu_seqlens[s], which is row place % page_size of page page_table[s, place / page_size].  A place is not a position:
a sequence that lost rows to `evict8` holds fewer than it has positions.  cu_seqlens [n_seqs + 1], held and page_table [n_seqs, width]
are int32 on the device; every place a call reads or writes needs its page, and rows behind the last sequence are left as they were.
The launches go to the current stream, allocate their scratch from torch's allocator and can be captured into CUDA graphs."""
from __future__ import annotations

from ctypes import c_float, c_void_p
from typing import Optional, Tuple

import torch

from ..csrc.build import load_kernel
from ._call import KernelError, check, code, ints, on_current_device, ptr, stream, want_f32, want_int32
from .attention import PAIRING, prefill_rows, prefill_usable, resident_ctas
from .gemm_tc import status_word

BLOCK = 16
MAX_HEAD_DIM = 256


def storage(n_pages: int, n_kv_heads: int, page_size: int, head_dim: int, device, weights: bool = False
            ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(codes, scales, weights or None) of an empty cache."""
    check_sizes(page_size, head_dim)
    return (torch.zeros((n_pages, 2, n_kv_heads, page_size, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn),
            torch.ones((n_pages, 2, n_kv_heads, page_size // BLOCK), dtype=torch.uint8, device=device),
            torch.zeros((n_pages, n_kv_heads, page_size), dtype=torch.float32, device=device) if weights else None)


def check_sizes(page_size: int, head_dim: int) -> None:
    if head_dim % 16 or not 16 <= head_dim <= MAX_HEAD_DIM:
        raise KernelError(f"the 8-bit cache takes head sizes 16, 32, …, {MAX_HEAD_DIM}; got {head_dim}")
    if page_size % BLOCK or page_size < BLOCK:
        raise KernelError(f"the 8-bit cache takes pages of a multiple of {BLOCK} rows; got {page_size}")


def _check_cache(codes, scales, weights, page_table, page_size, n_kv_heads, head_dim) -> None:
    pages = codes.shape[0]
    if codes.dtype != torch.float8_e4m3fn or tuple(codes.shape) != (pages, 2, n_kv_heads, page_size, head_dim):
        raise KernelError(f"8-bit cache: codes must be float8_e4m3fn [pages, 2, {n_kv_heads}, {page_size}, {head_dim}], got {codes.dtype} {tuple(codes.shape)}")
    if scales.dtype != torch.uint8 or tuple(scales.shape) != (pages, 2, n_kv_heads, page_size // BLOCK):
        raise KernelError(f"8-bit cache: scales must be uint8 [{pages}, 2, {n_kv_heads}, {page_size // BLOCK}], got {scales.dtype} {tuple(scales.shape)}")
    if weights is not None and (weights.dtype != torch.float32 or tuple(weights.shape) != (pages, n_kv_heads, page_size)):
        raise KernelError(f"8-bit cache: weights must be float32 [{pages}, {n_kv_heads}, {page_size}], got {weights.dtype} {tuple(weights.shape)}")
    if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[1] < 1:
        raise KernelError(f"8-bit cache: the page table must be int32 [sequences, pages], got {page_table.dtype} {tuple(page_table.shape)}")


def _check_step(cu_seqlens, held, page_table, what: str) -> int:
    n = page_table.shape[0]
    want_int32(cu_seqlens, "cu_seqlens")
    want_int32(held, "held")
    if cu_seqlens.numel() != n + 1 or held.numel() != n:
        raise KernelError(f"{what}: {n} page tables, {held.numel()} counts of held rows and {cu_seqlens.numel()} run borders do not fit together")
    return n


def write_rows8(qkv: torch.Tensor, bias: Optional[torch.Tensor], cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], pairing: str,
                positions: torch.Tensor, cu_seqlens: torch.Tensor, held: torch.Tensor, page_table: torch.Tensor, page_size: int,
                q_out: torch.Tensor, codes: Optional[torch.Tensor], scales: Optional[torch.Tensor], n_heads: int, n_kv_heads: int, head_dim: int,
                max_q_len: int) -> None:
    """Bias and rotary encoding (by positions [T]; cos and sin [positions, head_dim / 2] float32 or None) on the fused projection qkv
    [T, (nh + 2 nkv) * hd]; queries to q_out [T, nh, hd], keys and values as codes to their places (codes and scales None: the queries
    only, for layers that read another layer's cache).  max_q_len: the longest run."""
    T = qkv.shape[0]
    if (codes is None) != (scales is None):
        raise KernelError("write_rows8: codes and scales come together")
    if codes is None:
        check_sizes(page_size, head_dim)
    else:
        _check_cache(codes, scales, None, page_table, page_size, n_kv_heads, head_dim)
    n = _check_step(cu_seqlens, held, page_table, "write_rows8")
    want_int32(positions, "positions")
    if qkv.shape[1] != (n_heads + 2 * n_kv_heads) * head_dim or q_out.numel() != T * n_heads * head_dim or positions.numel() != T or q_out.dtype != qkv.dtype \
            or (bias is not None and bias.numel() != qkv.shape[1]):
        raise KernelError(f"write_rows8: projection {tuple(qkv.shape)} {qkv.dtype}, queries {tuple(q_out.shape)} {q_out.dtype} and {positions.numel()} positions do not fit together")
    if (cos is None) != (sin is None):
        raise KernelError("write_rows8: cos and sin tables come together")
    if cos is not None:
        want_f32(cos, "cos table")
        want_f32(sin, "sin table")
        if cos.shape[-1] != head_dim // 2 or cos.shape != sin.shape:
            raise KernelError(f"write_rows8: cos and sin tables must be [positions, {head_dim // 2}]")
    if T == 0:
        return
    on_current_device(qkv, q_out, codes, scales)
    check("cache8", load_kernel("cache8").tq_write8(
        ptr(qkv), code(qkv.dtype), ptr(bias), 0 if bias is None else code(bias.dtype), ptr(cos), ptr(sin), PAIRING[pairing], ptr(positions),
        ptr(cu_seqlens), ptr(held), ptr(page_table), page_table.shape[1], page_size, ptr(q_out), ptr(codes), ptr(scales),
        0 if codes is None else codes.shape[0], n, *ints(max_q_len, n_heads, n_kv_heads, head_dim), stream()))


def ranges_for(tiles: int, blocks: int, resident: int) -> int:
    """Ranges the keys of a tile of columns are cut into: as many as fill the CTAs the device runs at once, each of at least two blocks of
    16 keys for its four warps; with more tiles than that, the count (up to 8) whose last wave is fullest, and one from four waves on."""
    most = max(1, blocks // 8)
    if tiles <= resident:
        return max(1, min(most, resident // tiles))
    if tiles >= 4 * resident:
        return 1
    fill = lambda n: tiles * n / (-(-tiles * n // resident) * resident)
    return max(range(1, min(8, most) + 1), key=lambda n: (round(fill(n), 2), -n))


SCORE_BYTES = 1 << 28        # scratch a decode step may take for scores


def attention8(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, cu_seqlens: torch.Tensor, held: torch.Tensor,
               page_table: torch.Tensor, page_size: int, window: int, scale: float, out: torch.Tensor, n_heads: int, n_kv_heads: int,
               head_dim: int, max_q_len: int, max_kv_len: int, weights: Optional[torch.Tensor] = None,
               status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the step's queries q [T, nh, hd] over the pages (the step's own rows are in them already): a row sees its
    sequence's places up to its own (window > 0: the last `window` of them), scores times `scale`; out [T, nh * hd] in q's type.
    max_q_len: the longest run; max_kv_len: at least the longest held + run.
    weights: the softmax weights that each cached row receives from the step's rows, summed over a key/value head's query heads, are
    added to its sum; the sums of the step's own rows start with this step.
    status: the word in which the prompt kernel reports a wait that ran out (default: the device's, kernels.gemm_tc)."""
    T = q.shape[0]
    _check_cache(codes, scales, weights, page_table, page_size, n_kv_heads, head_dim)
    n = _check_step(cu_seqlens, held, page_table, "attention8")
    if q.numel() != T * n_heads * head_dim or out.numel() != q.numel() or out.dtype != q.dtype:
        raise KernelError(f"attention8: queries {tuple(q.shape)} {q.dtype} and output {tuple(out.shape)} {out.dtype} do not fit {n_heads} heads of {head_dim}")
    if T == 0 or n == 0 or max_q_len < 1:
        return out
    on_current_device(q, out, codes, scales, weights)
    if max_q_len >= PROMPT_MIN_RUN and prefill_usable(q.dtype, head_dim, page_size):
        return _attention8_prompt(q, codes, scales, cu_seqlens, held, page_table, page_size, window, scale, out, n_heads, n_kv_heads, head_dim,
                                  max_q_len, max_kv_len, weights, status)
    per = n_heads // n_kv_heads
    columns = max_q_len * per
    wide = columns > 8 and head_dim <= 128                  # two tiles of 8 columns in one CTA
    tiles = -(-columns // (16 if wide else 8)) * n_kv_heads * n
    per_sm = 2 if head_dim > 128 else 3 if wide and head_dim > 64 else 4         # CTAs an SM holds
    ranges = ranges_for(tiles, -(-max_kv_len // BLOCK), resident_ctas(q.device) // 4 * per_sm)
    # one row a sequence: the first launch leaves its scores for the second one to add up, which moves 8 bytes a key and query head, where
    # reading the keys again moves head_dim bytes a key
    stride = -(-max_kv_len // BLOCK) * BLOCK
    stored = weights is not None and max_q_len == 1 and 8 * per <= head_dim and 4 * T * n_heads * stride <= SCORE_BYTES
    rows = T * n_heads
    partial_floats = rows * ranges * (head_dim + 4) if ranges > 1 or stored else 0
    scratch = torch.empty(partial_floats + (rows * stride if stored else 0) + (rows if weights is not None and not stored else 0), dtype=torch.float32,
                          device=q.device) if weights is not None or partial_floats else None
    at = 0 if scratch is None else scratch.data_ptr()
    partial = at if partial_floats else None
    rest = at + 4 * partial_floats
    lib = load_kernel("attention8")
    args = (ptr(q), ptr(codes), ptr(scales), code(q.dtype), ptr(cu_seqlens), ptr(held), ptr(page_table), page_table.shape[1], *ints(page_size, window), c_float(scale))
    step = (codes.shape[0], n, *ints(max_q_len))
    heads = (*ints(n_heads, n_kv_heads, head_dim), stream())
    check("attention8", lib.tq_attention8(*args, ptr(out), c_void_p(partial), ranges, c_void_p(rest if weights is not None and not stored else None),
                                          c_void_p(rest if stored else None), stride, ptr(weights) if stored else None, *ints(max_kv_len), *step, *heads),
          kernels=2 if partial_floats else 1)
    if weights is not None and not stored:
        check("attention8", lib.tq_weigh8(*args, c_void_p(rest), ptr(weights), *step, *ints(max_kv_len), *heads))
    return out


PROMPT_MIN_RUN = 48          # steps whose longest run is at least this go to the tensor-core prompt kernel, where it takes their sizes
DENSE_BYTES = 1 << 30        # scratch a step may take for pages in bfloat16; sequences beyond it follow in further launches


def _attention8_prompt(q, codes, scales, cu_seqlens, held, page_table, page_size, window, scale, out, n_heads, n_kv_heads, head_dim, max_q_len,
                       max_kv_len, weights, status):
    """The pages a step sees are expanded to bfloat16 pages of a scratch, exactly, and the prompt kernel of csrc/attention_prefill.cu reads those."""
    T, n = q.shape[0], page_table.shape[0]
    if status is None:
        status = status_word(q.device)
    width = -(-max_kv_len // page_size)
    page_bytes = 2 * n_kv_heads * page_size * head_dim * 2
    group = max(1, min(n, DENSE_BYTES // (page_bytes * width)))
    dense = torch.empty((group * width, 2, n_kv_heads, page_size, head_dim), dtype=torch.bfloat16, device=q.device)
    table = torch.empty((group, width), dtype=torch.int32, device=q.device)
    lost = torch.empty((group, n_kv_heads, width), dtype=torch.uint8, device=q.device)
    lse = torch.empty((T, n_heads), dtype=torch.float32, device=q.device) if weights is not None else None
    for i in range(0, n, group):
        m = min(group, n - i)
        cu, starts, pages, dtable = cu_seqlens[i:i + m + 1], held[i:i + m], page_table[i:i + m], table[:m]
        cache = (ptr(codes), ptr(scales), ptr(cu), ptr(starts), ptr(pages), pages.shape[1], *ints(page_size, window))
        check("prompt8", load_kernel("prompt8").tq_expand8(*cache, ptr(dense), ptr(table), ptr(lost), width, codes.shape[0], m, *ints(n_kv_heads, head_dim), stream()))
        prefill_rows(q, dense, 2, cu, starts, dtable, page_size, window, scale, out, m, max_q_len, n_heads, n_kv_heads, head_dim, head_dim, status=status, lse=lse)
        check("attention8", load_kernel("attention8").tq_repair8(
            ptr(q), *cache, c_float(scale), ptr(out), ptr(lost), width, codes.shape[0], m, *ints(n_heads, n_kv_heads, head_dim), stream()))
        if weights is not None:
            check("prompt8", load_kernel("prompt8").tq_weigh8_prompt(
                ptr(q), ptr(dense), width, ptr(cu), ptr(starts), ptr(pages), pages.shape[1], *ints(window), c_float(scale), ptr(lse), ptr(weights),
                codes.shape[0], T, m, *ints(max_kv_len, n_heads, n_kv_heads, head_dim), ptr(status), stream()))
    return out


def evict8(codes: torch.Tensor, scales: torch.Tensor, weights: torch.Tensor, lengths: torch.Tensor, page_table: torch.Tensor,
           new_table: torch.Tensor, page_size: int, budget: int, recent: int) -> torch.Tensor:
    """Sequences of lengths [n_seqs] rows go to the pages of new_table [n_seqs, at least budget / page_size] and keep at most `budget`
    rows in each key/value head: the last `recent` and, of those before, the ones with the largest weights (the first of equal ones;
    NaN counts as the smallest), in the order of their places.  A sequence within the budget keeps all its rows.  A new block takes the
    largest byte of its rows, rows of a smaller one are rounded again; sums of weights move along.  The old pages are only read and must
    not be among the new ones; rows of the new pages behind a sequence's last stay as they were.  Returns the places that were kept,
    int32 [n_seqs, nkv, budget], -1 where there are fewer."""
    n_kv_heads, head_dim = codes.shape[2], codes.shape[4]
    _check_cache(codes, scales, weights, page_table, page_size, n_kv_heads, head_dim)
    check_sizes(page_size, head_dim)
    want_int32(lengths, "lengths")
    want_int32(new_table, "new page table")
    n = page_table.shape[0]
    if lengths.numel() != n or new_table.dim() != 2 or new_table.shape[0] != n or new_table.shape[1] * page_size < budget:
        raise KernelError(f"evict8: {n} page tables, {lengths.numel()} lengths and new tables {tuple(new_table.shape)} for a budget of {budget} rows do not fit together")
    if not 0 <= recent <= budget or budget < 1:
        raise KernelError(f"evict8: cannot keep the newest {recent} rows of a budget of {budget}")
    on_current_device(codes, scales, weights)
    kept = torch.empty((n, n_kv_heads, budget), dtype=torch.int32, device=codes.device)
    lib = load_kernel("evict")
    check("evict", lib.tq_evict8_select(
        ptr(weights), ptr(lengths), ptr(page_table), page_table.shape[1], *ints(page_size, codes.shape[0], n, n_kv_heads, budget, recent), ptr(kept), stream()))
    check("evict", lib.tq_evict8_move(
        ptr(codes), ptr(scales), ptr(weights), ptr(kept), ptr(page_table), page_table.shape[1], ptr(new_table), new_table.shape[1],
        *ints(page_size, codes.shape[0], n, n_kv_heads, head_dim, budget), stream()))
    return kept
