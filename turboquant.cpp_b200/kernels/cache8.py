"""A key/value cache in 8 bits whose length can be bounded (csrc/cache8.cu, csrc/attention8.cu, csrc/prompt8.cu, csrc/evict.cu).

An element is an e4m3 code times 2^(b - 127), b one byte for 16 consecutive rows of a (page, plane, key/value head): the smallest power of
two, of those from 2^-126 on, under which the largest finite magnitude of the 16 rows is at most 448.  A block that takes rows in
several steps keeps the largest byte; the rows it held are then rounded again.  What is not finite becomes NaN and does not count for the byte.

    codes    [pages, 2 (keys, values), kv heads, page_size, head size] float8_e4m3fn
    scales   [pages, 2, kv heads, page_size / 16] uint8
    weights  [pages, kv heads, page_size] float32: the attention weight each row has received, where it is kept

The step's rows are packed, sequence after sequence: rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1 belong to sequence s, and row t lies at
place held[s] + t - cu_seqlens[s], which is row place % page_size of page page_table[s, place / page_size].  A page belongs to one sequence of a call.  A place is not a position:
a sequence that lost rows to `evict8` holds fewer than it has positions.  cu_seqlens [n_seqs + 1], held and page_table [n_seqs, width]
are int32 on the device; every place a call reads or writes needs its page, and rows behind the last sequence are left as they were.
The launches go to the current stream, allocate their scratch from torch's allocator and can be captured into CUDA graphs."""
from __future__ import annotations

from functools import lru_cache
from operator import index
from typing import Optional, Tuple

import torch

from ..csrc.build import load_kernel
from ._call import KernelError, addresses, check, code, declared, packed, want_int32
from .attention import PAIRING, prefill_pieces, prefill_usable, resident_ctas
from .gemm_tc import status_word

BLOCK = 16
MAX_HEAD_DIM = 256


_PACKED = {"tq_write8": "12P11i", "tq_attention8": "12P13if", "tq_evict8": "8P9i"}        # members of the entry points' structs (_call.packed)
_SIGNATURES = {              # argument types of the others (_call.declared)
    "tq_weigh8": "pppippp" "iiifpp" "iiiiii" "p", "tq_repair8": "pppppp" "iiifppi" "iiiii" "p",
    "tq_expand8": "ppppp" "iiipppii" "iiii" "p", "tq_weigh8_prompt": "ppippp" "iifpp" "iiiiiii" "pp",
    "tq_attention_prefill": "ppippp" "iiiiii" "ffpippp" "iiiiiii" "pp", "tq_attention_prefill_split": "ppppp" "iiiifpppp" "iiiiiiii" "pp",
}
_entries = {}


def _declare(lib, name: str):
    fn = _entries[name] = packed(lib, name, _PACKED[name]) if name in _PACKED else declared(lib, name, _SIGNATURES[name])
    return fn


def _cache8(name: str):
    return _entries.get(name) or _declare(load_kernel("cache8"), name)


def _attention8(name: str):
    return _entries.get(name) or _declare(load_kernel("attention8"), name)


def _prompt8(name: str):
    return _entries.get(name) or _declare(load_kernel("prompt8"), name)


def _attention_prefill(name: str):
    return _entries.get(name) or _declare(load_kernel("attention_prefill"), name)


def _evict(name: str):
    return _entries.get(name) or _declare(load_kernel("evict"), name)


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


_E4M3, _U8, _F32, _I32 = torch.float8_e4m3fn, torch.uint8, torch.float32, torch.int32


def _sizes(codes, scales, weights, page_table, page_size: int, n_kv_heads: int, head_dim: int) -> Tuple[int, int, int]:
    """(pages, sequences, pages of a table) of a cache that fits together."""
    shape, table = codes.shape, page_table.shape
    pages = shape[0]
    if (shape == (pages, 2, n_kv_heads, page_size, head_dim) and codes.dtype is _E4M3 and scales.dtype is _U8
            and scales.shape == (pages, 2, n_kv_heads, page_size // BLOCK) and len(table) == 2 and page_table.dtype is _I32 and table[1] > 0
            and (weights is None or (weights.dtype is _F32 and weights.shape == (pages, n_kv_heads, page_size)))):
        return pages, table[0], table[1]
    if codes.dtype is not _E4M3 or shape != (pages, 2, n_kv_heads, page_size, head_dim):
        raise KernelError(f"8-bit cache: codes must be float8_e4m3fn [pages, 2, {n_kv_heads}, {page_size}, {head_dim}], got {codes.dtype} {tuple(shape)}")
    if scales.dtype is not _U8 or scales.shape != (pages, 2, n_kv_heads, page_size // BLOCK):
        raise KernelError(f"8-bit cache: scales must be uint8 [{pages}, 2, {n_kv_heads}, {page_size // BLOCK}], got {scales.dtype} {tuple(scales.shape)}")
    if weights is not None and (weights.dtype is not _F32 or weights.shape != (pages, n_kv_heads, page_size)):
        raise KernelError(f"8-bit cache: weights must be float32 [{pages}, {n_kv_heads}, {page_size}], got {weights.dtype} {tuple(weights.shape)}")
    raise _bad_table(page_table)


def _bad_table(page_table) -> KernelError:
    return KernelError(f"8-bit cache: the page table must be int32 [sequences, pages], got {page_table.dtype} {tuple(page_table.shape)}")


def _check_step(cu_seqlens, held, n: int, what: str) -> None:
    if not (cu_seqlens.dtype is _I32 and held.dtype is _I32 and cu_seqlens.numel() == n + 1 and held.numel() == n):
        want_int32(cu_seqlens, "cu_seqlens")
        want_int32(held, "held")
        raise KernelError(f"{what}: {n} page tables, {held.numel()} counts of held rows and {cu_seqlens.numel()} run borders do not fit together")


def write_rows8(qkv: torch.Tensor, bias: Optional[torch.Tensor], cos: Optional[torch.Tensor], sin: Optional[torch.Tensor], pairing: str,
                positions: torch.Tensor, cu_seqlens: torch.Tensor, held: torch.Tensor, page_table: torch.Tensor, page_size: int,
                q_out: torch.Tensor, codes: Optional[torch.Tensor], scales: Optional[torch.Tensor], n_heads: int, n_kv_heads: int, head_dim: int,
                max_q_len: int) -> None:
    """Bias and rotary encoding (by positions [T]; cos and sin [positions, head_dim / 2] float32 or None) on the fused projection qkv
    [T, (nh + 2 nkv) * hd]; queries to q_out [T, nh, hd], keys and values as codes to their places (codes and scales None: the queries
    only, for layers that read another layer's cache).  max_q_len: the longest run."""
    T, columns = qkv.shape
    if codes is None or scales is None:
        if codes is not None or scales is not None:
            raise KernelError("write_rows8: codes and scales come together")
        check_sizes(page_size, head_dim)
        if page_table.dtype is not _I32 or page_table.dim() != 2 or page_table.shape[1] < 1:
            raise _bad_table(page_table)
        pages, (n, width) = 0, page_table.shape
    else:
        pages, n, width = _sizes(codes, scales, None, page_table, page_size, n_kv_heads, head_dim)
    _check_step(cu_seqlens, held, n, "write_rows8")
    dtype = qkv.dtype
    if n_kv_heads < 1 or n_heads < 1 or n_heads % n_kv_heads:
        raise KernelError(f"write_rows8: {n_heads} heads are not a multiple of {n_kv_heads} key/value heads")
    if columns != (n_heads + 2 * n_kv_heads) * head_dim or q_out.numel() != T * n_heads * head_dim or q_out.dtype is not dtype \
            or positions.numel() != T or positions.dtype is not _I32 or (bias is not None and bias.numel() != columns):
        want_int32(positions, "positions")
        raise KernelError(f"write_rows8: projection {tuple(qkv.shape)} {dtype}, queries {tuple(q_out.shape)} {q_out.dtype} and {positions.numel()} positions do not fit together")
    if cos is not None or sin is not None:
        if cos is None or sin is None:
            raise KernelError("write_rows8: cos and sin tables come together")
        if cos.dtype is not _F32 or sin.dtype is not _F32 or cos.shape != sin.shape or cos.shape[-1] != head_dim // 2:
            raise KernelError(f"write_rows8: cos and sin tables must be float32 [positions, {head_dim // 2}]")
    if T == 0:
        return
    p_qkv, p_bias, p_cos, p_sin, p_positions, p_cu, p_held, p_table, p_q, p_codes, p_scales, at = addresses(
        qkv, bias, cos, sin, positions, cu_seqlens, held, page_table, q_out, codes, scales)
    check("cache8", _cache8("tq_write8")(
        p_qkv, p_bias, p_cos, p_sin, p_positions, p_cu, p_held, p_table, p_q, p_codes, p_scales, at,
        code(dtype), 0 if bias is None else code(bias.dtype), PAIRING[pairing], width, page_size, pages, n, max_q_len, n_heads, n_kv_heads, head_dim))


MAX_RANGES, CLUSTER = 64, 8
# what a CTA's begin and end, the join of a cluster and that of a second launch take, in turns of a CTA's warps over blocks of keys
SETUP, CLUSTER_JOIN, JOIN = 1.5, 1.0, 6.0


@lru_cache(maxsize=4096)
def ranges_for(tiles: int, blocks: int, resident: int) -> int:
    """Ranges the keys of a tile of columns are cut into, where the device runs `resident` CTAs at once and a CTA's four warps take a block of 16
    keys each in turn: the count with the fewest turns.  (B200, device time, 16 heads of 128, 64 sequences of up to 2,048 keys, 1,024 tiles: one
    range 80 us, two 94, three 100, four 108.)  `blocks` is what the call says its longest sequence holds: a captured step says the longest there could be and
    is cut for that (these 64 planned for 8,192 keys: four ranges, 108 us; one of 700 rows 9.6 us where 6 ranges take 6.2; 32 of
    4,096 rows, seven query heads on a key/value head, with sums: no difference)."""
    turns = lambda n: -(-tiles * n // resident) * (-(-blocks // (4 * n)) + SETUP) + (0.0 if n == 1 else CLUSTER_JOIN if n <= CLUSTER else JOIN)
    most = max(1, min(MAX_RANGES, blocks // 4, max(CLUSTER, resident // tiles)))
    return min((n for n in (1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 24, 32, 48, most) if n <= most), key=lambda n: (turns(n), n))


_multiprocessors = {}


def _sms(t: torch.Tensor) -> int:
    """SMs of a tensor's device."""
    i = t.get_device()
    if i not in _multiprocessors:
        _multiprocessors[i] = resident_ctas(t.device) // 4
    return _multiprocessors[i]


SCORE_BYTES = 1 << 28        # scratch a decode step may take for scores


def attention8(q: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, cu_seqlens: torch.Tensor, held: torch.Tensor,
               page_table: torch.Tensor, page_size: int, window: int, scale: float, out: torch.Tensor, n_heads: int, n_kv_heads: int,
               head_dim: int, max_q_len: int, max_kv_len: int, weights: Optional[torch.Tensor] = None,
               status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the step's queries q [T, nh, hd] over the pages (the step's own rows are in them already): a row sees its
    sequence's places up to its own (window > 0: the last `window` of them), scores times `scale`; out [T, nh * hd] in q's type.
    max_q_len: the longest run; max_kv_len: at least the longest held + run.  Large steps of bfloat16 with heads of 64 or 128 take scratch for the pages
    they see in bfloat16: up to DENSE_BYTES, or one sequence's.
    weights: the softmax weights that each cached row receives from the step's rows, summed over a key/value head's query heads, are
    added to its sum; the sums of the step's own rows start with this step.
    status: the word in which the prompt kernel reports a wait that ran out (default: the device's, kernels.gemm_tc)."""
    T, dtype = q.shape[0], q.dtype
    pages, n, width = _sizes(codes, scales, weights, page_table, page_size, n_kv_heads, head_dim)
    _check_step(cu_seqlens, held, n, "attention8")
    if n_kv_heads < 1 or n_heads < 1 or n_heads % n_kv_heads:
        raise KernelError(f"attention8: {n_heads} heads are not a multiple of {n_kv_heads} key/value heads")
    elements = T * n_heads * head_dim
    if q.numel() != elements or out.numel() != elements or out.dtype is not dtype:
        raise KernelError(f"attention8: queries {tuple(q.shape)} {dtype} and output {tuple(out.shape)} {out.dtype} do not fit {n_heads} heads of {head_dim}")
    if T == 0 or n == 0 or max_q_len < 1:
        return out
    max_q_len, max_kv_len = index(max_q_len), index(max_kv_len)
    if max_q_len >= PROMPT_MIN_RUN and prefill_usable(dtype, head_dim, page_size) and T * (max_kv_len - max_q_len // 2) * n_heads * head_dim >= PROMPT_WORK:
        # the prompt kernel copies and stores 16 bytes at a time: queries and results that begin elsewhere go through a copy
        if q.is_contiguous() and q.data_ptr() % 16:
            q = q.clone()
        to = out.clone() if out.is_contiguous() and out.data_ptr() % 16 else out           # (rows behind the last sequence come back as they were)
        _attention8_prompt(q, codes, scales, cu_seqlens, held, page_table, page_size, window, scale, to, n_heads, n_kv_heads, head_dim,
                           max_q_len, max_kv_len, weights, status)
        return out if to is out else out.copy_(to)
    p_q, p_out, p_codes, p_scales, p_cu, p_held, p_table, p_weights, at = addresses(q, out, codes, scales, cu_seqlens, held, page_table, weights)
    per = n_heads // n_kv_heads
    columns = max_q_len * per
    wide = columns > 8 and head_dim <= 128                  # two tiles of 8 columns in one CTA
    own_tiles = -(-columns // (16 if wide else 8))          # of a sequence and key/value head
    per_sm = 2 if head_dim > 128 else 3 if wide and head_dim > 64 else 4         # CTAs an SM holds
    blocks = -(-max_kv_len // BLOCK)
    ranges = ranges_for(own_tiles * n_kv_heads * n, blocks, _sms(q) * per_sm)
    partial = again = scores = stride = 0
    joins = ranges > CLUSTER                                # in a second launch
    if weights is not None:
        # one row a sequence: scores are left for whoever joins the ranges, to be added up, which moves 8 bytes a key and query head, where reading
        # the keys again moves head_dim bytes a key
        stride, rows = blocks * BLOCK, T * n_heads
        size = n * n_kv_heads * stride * (per if per <= 2 else 4 if per <= 4 else 8 if per <= 8 else -(-per // 16) * 16)
        stored = max_q_len == 1 and 8 * per <= head_dim and 4 * size <= SCORE_BYTES
        joins |= stored and (ranges == 1 or own_tiles > 1)
        sums = rows * ranges * (head_dim + 4) if joins else 0
        scratch = torch.empty(sums + (size if stored else rows), dtype=torch.float32, device=q.device)
        partial = scratch.data_ptr() if joins else 0
        if stored:
            scores = scratch.data_ptr() + 4 * sums
        else:
            again = scratch.data_ptr() + 4 * sums           # the rows' denominators, for a launch that reads the keys again
    elif joins:
        scratch = torch.empty(T * n_heads * ranges * (head_dim + 4), dtype=torch.float32, device=q.device)
        partial = scratch.data_ptr()
    kind = code(dtype)
    check("attention8", _attention8("tq_attention8")(
        p_q, p_codes, p_scales, p_cu, p_held, p_table, p_out, partial, again, scores, p_weights if scores else 0, at,
        kind, width, page_size, window, ranges, stride, max_kv_len, pages, n, max_q_len, n_heads, n_kv_heads, head_dim, scale), kernels=2 if joins else 1)
    if again:
        check("attention8", _attention8("tq_weigh8")(
            p_q, p_codes, p_scales, kind, p_cu, p_held, p_table, width, page_size, window, scale, again, p_weights, pages, n, max_kv_len,
            n_heads, n_kv_heads, head_dim, at))
    return out


# Steps whose longest run is at least this, and whose queries, heads, elements and the keys they see multiply to this much, go to the tensor-core
# prompt kernel, where it takes their sizes.  (B200, us, csrc/attention8.cu and the prompt kernel's five launches: 128 rows behind 800, 16
# heads of 128, 0.2e9: 19 and 31; 28 heads on 4, 0.4e9: 39 and 31; 64 behind 4,000, 16 heads, 0.5e9: 28 and 38; 128 behind 4,000, 1.1e9: 44 and 40;
# 256 behind 4,000, 2.2e9: 119 and 46.)  A window is left out of the count: behind 30,000 with a window of 128, 64 rows, 16 heads: 14 and 23, 28 on 4: 30 and
# 17; 512 rows: 103 and 31, 231 and 26.
PROMPT_MIN_RUN, PROMPT_WORK = 48, 350_000_000
DENSE_BYTES = 1 << 30        # scratch a step may take for pages in bfloat16 (or one sequence's, if they are more); sequences beyond it follow in further launches


def _attention8_prompt(q, codes, scales, cu_seqlens, held, page_table, page_size, window, scale, out, n_heads, n_kv_heads, head_dim, max_q_len,
                       max_kv_len, weights, status):
    """The pages a step sees are expanded to bfloat16 pages of a scratch, exactly, and the prompt kernel of csrc/attention_prefill.cu reads those."""
    T, (n, columns), pages = q.shape[0], page_table.shape, codes.shape[0]
    if status is None:
        status = status_word(q.device)
    p_q, p_out, p_codes, p_scales, p_cu, p_held, p_table, p_weights, p_status, at = addresses(
        q, out, codes, scales, cu_seqlens, held, page_table, weights, status)
    width = -(-max_kv_len // page_size)
    page_bytes = 2 * n_kv_heads * page_size * head_dim * 2
    dense_width = min(width, (window + max_q_len - 2) // page_size + 2) if window > 0 else width         # pages a sequence's rows see
    group = max(1, min(n, DENSE_BYTES // (page_bytes * dense_width)))
    pieces, piece_pages = prefill_pieces(T, group, max_q_len, max_kv_len, n_heads, n_kv_heads, head_dim, window, _sms(q)) if scale > 0.0 else (1, 0)
    # one allocation: the pages, the rows' denominators and the pieces' results (float32), the page table (int32), the pages' marks (bytes)
    rows = T * n_heads
    sizes = (group * dense_width * page_bytes, 4 * rows if weights is not None else 0, 4 * rows * pieces * (head_dim + 1) if pieces > 1 else 0, 4 * group * width,
             group * n_kv_heads * width)
    scratch = torch.empty(sum(sizes) + 64, dtype=torch.uint8, device=q.device)
    dense = scratch.data_ptr()
    lse = dense + sizes[0]
    part = -(-(lse + sizes[1]) // 16) * 16
    tables = part + sizes[2]
    lost = tables + sizes[3]
    p_lse = lse if weights is not None else 0
    for i in range(0, n, group):
        m, cu, starts, own = min(group, n - i), p_cu + 4 * i, p_held + 4 * i, p_table + 4 * i * columns
        cache = (p_codes, p_scales, cu, starts, own, columns, page_size, window)
        check("prompt8", _prompt8("tq_expand8")(*cache, dense, tables, lost, width, dense_width, pages, m, n_kv_heads, head_dim, at))
        if pieces > 1:
            check("attention_prefill", _attention_prefill("tq_attention_prefill_split")(
                p_q, dense, cu, starts, tables, width, page_size, group * dense_width, window, scale, p_out, p_lse, part, part + 4 * rows * pieces * head_dim,
                pieces, piece_pages, T, m, max_q_len, n_heads, n_kv_heads, head_dim, p_status, at), kernels=2)
        else:
            check("attention_prefill", _attention_prefill("tq_attention_prefill")(
                p_q, dense, 2, cu, starts, tables, width, page_size, group * dense_width, window, 0, 0, scale, 0.0, 0, 0, 0, p_out, p_lse, T, m, max_q_len,
                n_heads, n_kv_heads, head_dim, head_dim, p_status, at))
        check("attention8", _attention8("tq_repair8")(p_q, *cache, scale, p_out, lost, width, pages, m, n_heads, n_kv_heads, head_dim, at))
        if weights is not None:
            check("prompt8", _prompt8("tq_weigh8_prompt")(
                p_q, dense, dense_width, cu, starts, own, columns, window, scale, p_lse, p_weights, pages, T, m, max_kv_len,
                n_heads, n_kv_heads, head_dim, p_status, at))
    return out


def evict8(codes: torch.Tensor, scales: torch.Tensor, weights: torch.Tensor, lengths: torch.Tensor, page_table: torch.Tensor,
           new_table: torch.Tensor, page_size: int, budget: int, recent: int) -> torch.Tensor:
    """Sequences of lengths [n_seqs] rows go to the pages of new_table [n_seqs, at least budget / page_size] and keep at most `budget`
    rows in each key/value head: the last `recent` and, of those before, the ones with the largest weights (the first of equal ones;
    NaN counts as the smallest), in the order of their places.  A sequence within the budget keeps all its rows.  A new block takes the
    largest byte of its rows, rows of a smaller one are rounded again; sums of weights move along.  The old pages are only read and must
    not be among the new ones; rows of the new pages behind a sequence's last stay as they were; weights start on a 16-byte boundary.
    Returns the places that were kept, int32 [n_seqs, nkv, budget], -1 where there are fewer."""
    if codes.dim() != 5:
        raise KernelError(f"8-bit cache: codes must be float8_e4m3fn [pages, 2, kv heads, page_size, head size], got {tuple(codes.shape)}")
    if weights is None:
        raise KernelError("evict8: a cache without sums of weights has nothing to choose rows by")
    _, _, n_kv_heads, _, head_dim = codes.shape
    pages, n, width = _sizes(codes, scales, weights, page_table, page_size, n_kv_heads, head_dim)
    check_sizes(page_size, head_dim)
    if lengths.dtype is not _I32 or new_table.dtype is not _I32 or lengths.numel() != n or new_table.dim() != 2 or new_table.shape[0] != n \
            or new_table.shape[1] * page_size < budget:
        want_int32(lengths, "lengths")
        want_int32(new_table, "new page table")
        raise KernelError(f"evict8: {n} page tables, {lengths.numel()} lengths and new tables {tuple(new_table.shape)} for a budget of {budget} rows do not fit together")
    if not 0 <= recent <= budget or budget < 1:
        raise KernelError(f"evict8: cannot keep the newest {recent} rows of a budget of {budget}")
    p_codes, p_scales, p_weights, p_lengths, p_table, p_new, at = addresses(codes, scales, weights, lengths, page_table, new_table)
    kept = torch.empty((n, n_kv_heads, budget), dtype=torch.int32, device=codes.device)
    check("evict", _evict("tq_evict8")(
        p_codes, p_scales, p_weights, p_lengths, p_table, p_new, kept.data_ptr(), at, width, new_table.shape[1], page_size, pages, n, n_kv_heads, head_dim,
        budget, recent), kernels=2)
    return kept
