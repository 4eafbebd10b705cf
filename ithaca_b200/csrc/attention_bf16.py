"""Attention kernels of the bfloat16 path: one compiled module per head size.

``attention_bf16.cu`` is specialised at compile time for a head size; the module for the
size a model has is compiled the first time that model runs a step (a few seconds) and kept
beside the core library.
"""
from __future__ import annotations

import ctypes
from typing import Dict, Optional, Tuple

import torch

from . import build
from . import ops
from .ops import KernelError, _check, _ptr, _stream, sm_count

_vp, _i, _f = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
_modules: Dict[tuple, ctypes.CDLL] = {}

# Modules with options, measured on B200 (head sizes 64 and 128, contexts 2k-8k, batches 8-64): a ring of 60 KB a block leaves room for
# enough blocks per SM; where heads stop early the blocks of a sequence are unequal, and chunks of at most 8 pages even them out.
OPTION_RING_KB, REACH_CHUNK_PAGES = 60, 8
DECODE_CHUNK_PAGES = 4        # default: a decode block covers 4 pages = 256 keys; chunks start at multiples of that


def decode_chunk_pages(n_seqs: int, n_heads: int, n_kv_heads: int, max_kv_len: int, page_size: int = 64,
                       n_sm: Optional[int] = None) -> int:
    """Pages per decode block.  Measured on B200 (head size 128, 8 kv heads, contexts 1k-16k, batches 1-64,
    chunks of 2-32 pages): the kernel is fastest with about two blocks per SM in ONE wave, so the pages of a
    sequence are cut into as many chunks as that allows, but into chunks of at least 4 pages (2 when even
    that leaves most SMs idle: set-up and merging per block cost about as much as reading two pages).  With
    more (sequence, kv head) groups than two per SM, or a count that would load the SMs unevenly, there
    are several waves anyway; a long chunk and a short rest then pack best (the short blocks of the last chunk
    start last and fill the tail).  Over 72 measured (batch, context) pairs the chunk picked here is within 1 % of
    the best one's time on average, 13 % at worst."""
    N_SM = n_sm if n_sm is not None else sm_count()
    groups = n_seqs * n_kv_heads * -(-(n_heads // n_kv_heads) // 16)
    pages = max(1, -(-max_kv_len // page_size))
    if groups <= N_SM or groups > 1.5 * N_SM and groups <= 2 * N_SM:
        # (between one and one and a half groups per SM a single wave would give some SMs two blocks and others one)
        n_chunks = max(1, (2 * N_SM) // groups)
        least = 4 if groups * -(-pages // 4) >= 128 else 2
        return min(pages, max(-(-pages // n_chunks), least))
    return -(-pages * 3 // 4) if pages <= 24 else 20


def decode_chunk_pages_uneven(pages, n_heads: int, n_kv_heads: int, chunk: int, n_sm: int) -> int:
    """Pages per decode block for sequences of so many ``pages`` each, ``chunk`` being what would suit them all as long as the longest.  Where they come
    to less than 85 % of that, blocks are fewer and longer than the SMs want.  Then the shortest chunk of up to 12 pages that makes at most three
    blocks per SM and 18 pieces of a sequence (more cost more to merge than they gain); where there are more blocks whatever the chunk, 12 pages if the
    sequences differ by more, and nothing shorter where there are so many sequences and kv heads that they fill the SMs anyway.
    us on B200, lengths between a quarter and all of the longest, ``chunk`` / this, 32 heads of 128 on 8 kv heads: 8 sequences up to 4,000 30.4 / 21.0, 16 of 3,000
    41.5 / 28.0, 10 of 6,000 53.7 / 34.3, 20 of 600 18.4 / 15.0, 3 of 8,000 24.2 / 23; 40 heads on 40: 3 of 8,000 97 / 65, 8 of 4,000 79 / 70; one of 8,000 beside 15 of
    500 74 / 26."""
    n, most, total = len(pages), max(pages), sum(pages)
    if n < 2 or total >= 0.85 * n * most:
        return chunk
    groups = n_kv_heads * -(-(n_heads // n_kv_heads) // 16)
    if n * groups > 2.4 * n_sm:
        return min(12, chunk) if total < 0.35 * n * most else chunk
    least = max(2, -(-most // 18))
    for c in range(least, max(13, least + 1)):
        if sum(-(-p // c) for p in pages) * groups <= 3 * n_sm:
            return c if c <= 0.8 * chunk else chunk
    return min(12, chunk) if total < 0.75 * n * most else chunk


def seen_pages(kv_len_bound: int, window: int, keep: int, page_size: int = 64) -> int:
    """The most pages a query of a sequence of up to ``kv_len_bound`` positions sees: all, or under a window (> 0) those of
    the first ``keep`` keys and those a window of that many keys can reach into."""
    pages = max(1, -(-kv_len_bound // page_size))
    if window <= 0:
        return pages
    return min(pages, -(-keep // page_size) + (window + page_size - 2) // page_size + 1)


def supported(head_dim: int) -> bool:
    return head_dim % 16 == 0 and 16 <= head_dim <= 256


def module(head_dim: int, slopes: bool = False, one_row: bool = False) -> ctypes.CDLL:
    """The module of a head size; ``slopes``: with a distance bias, ``one_row``: for pages whose rows are keys and values."""
    key = (head_dim, slopes, one_row)
    m = _modules.get(key)
    if m is None:
        m = build.load_library(*build.attention_module(head_dim, slopes, one_row))
        m.ik_attn_prefill.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _f, _f, _i, _i, _i, _vp, _vp, _vp, _f, _f, _i, _i, _i, _vp, _vp]
        m.ik_attn_prefill.restype = _i
        m.ik_attn_prefill_tc.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _i, _f, _f, _i, _i, _i, _vp, _vp, _vp, _f, _f, _i, _i, _i, _vp, _vp]
        m.ik_attn_prefill_tc.restype = _i
        m.ik_attn_prefill_two_heads.argtypes = m.ik_attn_prefill_tc.argtypes
        m.ik_attn_prefill_two_heads.restype = _i
        m.ik_attn_decode.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _f, _f, _i, _i, _i, _vp, _vp, _vp, _f, _f, _i, _i, _i, _i, _i, _i,
                                     _vp, _vp]
        m.ik_attn_decode.restype = _i
        m.ik_attn_take_wait_record.argtypes = [_vp]
        m.ik_attn_take_wait_record.restype = _i
        if m.ik_attn_head_dim() != head_dim:
            raise KernelError("the attention module was compiled for another head size")
        _modules[key] = m
    return ops.timed(m)


def prefill(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, cu_seqlens: torch.Tensor,
            kv_lens: torch.Tensor, table: torch.Tensor, n_seqs: int, max_new: int, n_heads: int, scale: float,
            window: int, status: Optional[torch.Tensor], out: Optional[torch.Tensor] = None,
            kind: str = "auto", work: Optional[Tuple[int, int]] = None, softcap: float = 0.0, sink=False, keep: int = 0,
            key_scales: Optional[torch.Tensor] = None, slopes: Optional[torch.Tensor] = None, reach=None,
            two_heads: bool = False) -> torch.Tensor:
    """``kind``: "tc" = the tcgen05 kernel (head sizes 64 and 128), "two_heads" = the one with two heads a block, "mma" = the
    warp-level kernel, "auto" = tcgen05 where it applies (``two_heads``: with two heads a block where that kernel takes the call).  ``softcap``: scores become cap * tanh(score / cap) (0 = no cap).  ``sink``: the
    softmax's denominator counts one more key of score 0 that carries no value (True), or of a score per head (a float32
    tensor [n_heads], not scaled).  ``key_scales``: the pages' rows are keys and values (``v_pages`` None), and every score is
    multiplied by its key's number.  ``slopes`` [n_heads]: a score loses slope * distance, behind the cap.  ``reach`` = (norm, coef, every): no
    score in front of cap and bias is larger than norm * |1 + coef ln(floor((pos + 1) / every) + 1)| (every 0: than norm), so that keys
    the bias makes negligible need not be visited (None: nothing is known).  ``keep``: under a window the first ``keep`` keys stay visible."""
    n_pages, nkv, page_size, hd = k_pages.shape
    ops.check_score_extras(key_scales, slopes, k_pages, n_heads)
    m = module(hd, slopes is not None, key_scales is not None)
    if out is None:
        out = torch.empty_like(q)
    ways = [kind] if kind in ("tc", "two_heads") else []
    if kind == "auto" and hd in (64, 128):
        ways = ["two_heads", "tc"] if two_heads else ["tc"]
    for way in ways:
        ops._work(f"attention prefill tcgen05 {q.shape[0]}x{n_heads}", *(work or (0, 0)))
        st = (m.ik_attn_prefill_two_heads if way == "two_heads" else m.ik_attn_prefill_tc)(_ptr(q), _ptr(k_pages), _ptr(v_pages), _ptr(out), _ptr(cu_seqlens), _ptr(kv_lens),
                                  _ptr(table), table.stride(0), q.shape[0], n_seqs, max_new, n_heads, nkv, scale, softcap, window, keep,
                                  ops.sink_flag(sink), _ptr(ops.sink_values(sink, n_heads)), _ptr(key_scales), _ptr(slopes), *(reach or (0.0, 0.0, 0)), page_size, n_pages, _ptr(status), _stream())
        if st != -2:
            _check(st, "attention prefill (tcgen05)")
            return out
    if kind in ("tc", "two_heads"):
        raise KernelError("attention prefill (tcgen05): head size or alignment not supported")
    ops._work(f"attention prefill mma {q.shape[0]}x{n_heads}", *(work or (0, 0)))
    _check(m.ik_attn_prefill(_ptr(q), _ptr(k_pages), _ptr(v_pages), _ptr(out), _ptr(cu_seqlens), _ptr(kv_lens),
                             _ptr(table), table.stride(0), n_seqs, max_new, n_heads, nkv, scale, softcap, window, keep, ops.sink_flag(sink),
                             _ptr(ops.sink_values(sink, n_heads)), _ptr(key_scales), _ptr(slopes), *(reach or (0.0, 0.0, 0)), page_size, n_pages, _ptr(status), _stream()), "attention prefill")
    return out


# Per head size and kernel (one head a block, two): us of a block besides its keys (with a window: more), per step of 64 or 128 keys
# beside other blocks and alone, of a block whose tile a shorter sequence does not have, the share of a whole round that a last round
# of equal blocks costs, of a launch, and the share of the longest block that unequal sequences add.
_Ways = Tuple[float, float, float, float, float, float, float, float]
PREFILL_COSTS: Dict[int, Tuple[_Ways, _Ways]] = {
    64: ((4.75, 1.37, 1.028, 0.743, 1.64, 0.80, 4.31, 0.27), (7.04, 2.39, 1.722, 1.594, 0.90, 1.06, 3.65, 0.05)),
    128: ((6.04, 1.96, 1.086, 0.757, 1.56, 0.70, 4.58, 0.30), (8.51, 2.67, 2.051, 1.907, 0.74, 1.03, 2.63, 0.09))}


def two_heads_pay(n_new, kv_lens, n_heads: int, hd: int, window: int, n_sm: int) -> bool:
    """Whether the prompts of a step run two heads a block (prompts without options, an even number of heads per kv head).

    Such a block has an SM to itself; of those with one head an SM holds two, and there are twice as many.  So two heads pay where
    tiles of 128 queries see many keys, and lose where they see few (short prompts, windows) or where the last round of the SMs is nearly
    empty.  The times of both are estimated from the tiles that exist; the estimates' figures are fitted to measurements, 5 to 7 % off.
    Measured on B200 (us, one head / two; 32 heads on 8), heads of 128 and of 64: one prompt of 1,024 23 / 27 and 21 / 23, of 2,048 52 / 49 and
    49 / 42, of 4,096 148 / 143 and 134 / 121; 24 of 100 28 / 33 and 25 / 29, 64 of 130 124 / 168 and 104 / 139, eight of 1,000 114 / 128 and
    98 / 105, six of 50 to 2,000 134 / 118 and 112 / 92; 4,096 under a window of 128 52 / 63 and 45 / 56, of 1,024 94 / 97 and 84 / 85;
    512 behind 3,000 54 / 66 and 51 / 57."""
    counts = {}                                                     # tiles by the pages they see
    n_tiles = most = 0
    for n, e in zip(n_new, kv_lens):
        most = max(most, -(-n // 128))
        for lo in range(e - n, e, 128):
            pages = (min(lo + 128, e) - 1) // 64 - (max(0, lo + 1 - window) // 64 if window else 0) + 1
            counts[pages] = counts.get(pages, 0) + 1
            n_tiles += 1
    if not n_tiles:
        return False
    missing = most * len(n_new) - n_tiles

    def time(heads, slots, step_pages, costs):
        base, windowed, step, alone, none, last, launch, uneven = costs
        base += windowed if window else 0.0
        mean = base + step * sum(-(-p // step_pages) * c for p, c in counts.items()) / n_tiles
        top = -(-max(counts) // step_pages)
        longest = base + alone * top
        rounds = n_tiles * heads / slots
        us = longest
        if n_tiles * heads > n_sm:
            us = max(longest, mean * (rounds + last * (mean / (base + step * top)) ** 3 * (-(-n_tiles * heads // slots) - rounds)))
        return us + none * heads * missing / slots + uneven * longest * min(1.0, 2.5 * missing / n_tiles) + launch

    # near a tie two heads of 64 come out 2 % too cheap, and two of 128 4 % too dear for a prompt alone
    one, two = PREFILL_COSTS[hd]
    return time(n_heads // 2, n_sm, 2, two) < (0.98 if hd == 64 else 1.04 if len(n_new) == 1 else 1.0) * time(n_heads, 2 * n_sm, 1, one)


def _two_heads_of(ctx, n_heads: int, hd: int, window: int) -> bool:
    """``two_heads_pay`` of a step, once for all its layers of one kind."""
    key = ("two_heads_pay", n_heads, hd, window)
    if key not in ctx.shared:
        ctx.shared[key] = two_heads_pay(ctx.host_n_new, ctx.host_kv_lens, n_heads, hd, window, ops.sm_count())
    return ctx.shared[key]


def decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, kv_lens: torch.Tensor, table: torch.Tensor,
           n_seqs: int, kv_len_bound: int, n_heads: int, scale: float, window: int, status: Optional[torch.Tensor],
           out: Optional[torch.Tensor] = None, chunk_pages: int = DECODE_CHUNK_PAGES, ring_kb: int = 0,
           work: Optional[Tuple[int, int]] = None, softcap: float = 0.0, sink=False, keep: int = 0,
            key_scales: Optional[torch.Tensor] = None, slopes: Optional[torch.Tensor] = None, reach=None) -> torch.Tensor:
    """``kv_len_bound``: no sequence of the step is longer than this (it sizes the grid and the
    scratch for the partial results; blocks beyond a sequence's length return at once).  ``keep``: under a window the
    first ``keep`` keys stay visible."""
    n_pages, nkv, page_size, hd = k_pages.shape
    ops.check_score_extras(key_scales, slopes, k_pages, n_heads)
    m = module(hd, slopes is not None, key_scales is not None)
    n_splits = max(1, -(-seen_pages(kv_len_bound, window, keep, page_size) // chunk_pages))
    part_o = torch.empty((n_seqs, n_heads, n_splits, hd), dtype=torch.float32, device=q.device)
    part_ml = torch.empty((n_seqs, n_heads, n_splits, 2), dtype=torch.float32, device=q.device)
    if out is None:
        out = torch.empty_like(q)
    ops._work(f"attention decode {n_seqs}x{n_heads}", *(work or (0, 0)))
    _check(m.ik_attn_decode(_ptr(q), _ptr(k_pages), _ptr(v_pages), _ptr(out), _ptr(part_o), _ptr(part_ml),
                            _ptr(kv_lens), _ptr(table), table.stride(0), n_seqs, n_heads, nkv, scale, softcap, window, keep,
                            ops.sink_flag(sink), _ptr(ops.sink_values(sink, n_heads)), _ptr(key_scales), _ptr(slopes), *(reach or (0.0, 0.0, 0)), page_size, n_pages, chunk_pages, n_splits, ring_kb,
                            _ptr(status), _stream()), "attention decode", kernels=2)
    return out


_shared_modules: Dict[int, ctypes.CDLL] = {}
_shared_scratch: Dict[tuple, int] = {}         # bytes of scratch by device and sizes


def shared_module(head_dim: int) -> ctypes.CDLL:
    """The module of a head size for sequences that share pages."""
    m = _shared_modules.get(head_dim)
    if m is None:
        m = build.load_library(*build.shared_module(head_dim))
        m.ik_attn_shared.argtypes = [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _i, _vp, _vp, _i, _i, _i, _i, _i, _f, _f, _i, _vp, _i, _i, _vp, _vp]
        m.ik_attn_shared.restype = _i
        m.ik_attn_shared_scratch.argtypes, m.ik_attn_shared_scratch.restype = [_i, _i, _i, _i, _i], ctypes.c_longlong
        m.ik_attn_shared_take_wait_record.argtypes, m.ik_attn_shared_take_wait_record.restype = [_vp], _i
        if m.ik_attn_shared_head_dim() != head_dim:
            raise KernelError("the attention module was compiled for another head size")
        _shared_modules[head_dim] = m
    return ops.timed(m)


SHARED_SEQS_MOST = SHARED_TILES_MOST = 1024          # what one launch of the kernel for shared pages takes


def sharing_pays(n_seqs: int, n_groups: int, max_members: int, shared_bound: int, own_bound: int, n_heads: int, n_kv_heads: int, hd: int) -> bool:
    """Whether a decode step whose sequences share pages reads them once per group (``decode_shared``), from the sizes that a captured step is kept under.

    It saves (n_seqs - n_groups) readings of the shared pages per kv head, and costs 1 to 3 us more to set up; with more than 32 rows to a tile pages of one's own cost
    more there, too (all warps pass them, few have work).  us on B200, ``decode`` / ``decode_shared``, pages shared + own: 32 heads of 128 on 8, one group of 4: 8+1 9.1 / 9.3,
    16+1 11.2 / 9.9, 48+1 16.5 / 11.3; four of 2: 4+1 9.5 / 8.6, 8+1 11.3 / 9.6; four of 8: 2+1 10.9 / 11.7, 4+1 13.8 / 12.0, 2+4 15.4 / 18.7, 4+4 18.2 / 16.1; four of 16:
    2+1 18.6 / 15.7, 4+4 29.5 / 33.2, 8+4 38.9 / 27.9; sixteen of 4: 1+4 23.7 / 21.3, 48+4 127 / 55; 40 heads on 40, four of 16: 48+1 529 / 61.  32 heads of 64: one
    group of 4: 16+1 9.1 / 8.8; four of 4: 4+1 8.6 / 8.8, 8+1 10.1 / 9.2.  Over 396 such combinations the choice is 0.5 % behind the better one on average, 23 % at worst."""
    rows = max_members * (n_heads // n_kv_heads)
    tall = 16 if rows <= 16 else 32 if rows <= 32 else 64
    heads = min(n_heads // n_kv_heads, tall)
    tiles = n_groups * -(-max_members // max(1, min(tall // heads, max_members))) * -(-(n_heads // n_kv_heads) // heads)
    if n_seqs > SHARED_SEQS_MOST or tiles > SHARED_TILES_MOST:
        return False
    least, each = {16: (224, 0.0), 32: (512, 0.0), 64: (512, 0.75)}[tall]
    saved, own = (n_seqs - n_groups) * shared_bound * n_kv_heads, n_seqs * own_bound * n_kv_heads
    return saved * (hd + 64) / 192 >= least + each * own


def decode_shared(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, kv_lens: torch.Tensor, table: torch.Tensor, starts: torch.Tensor,
                  shared: torch.Tensor, n_groups: int, max_members: int, shared_bound: int, own_bound: int, n_heads: int, scale: float,
                  status: Optional[torch.Tensor], out: Optional[torch.Tensor] = None, softcap: float = 0.0, sink=False,
                  work: Optional[Tuple[int, int]] = None) -> torch.Tensor:
    """Attention of one new token per sequence (``q`` [B, heads * size], bfloat16) over pages of which groups of sequences share the first ones.  ``starts`` int32
    [n_groups + 1]: group g are the sequences starts[g] <= b < starts[g + 1], at most ``max_members`` of them (else ``status`` is set, and those beyond get zeros); ``shared`` int32 [B]: how many of sequence b's first pages are
    the same (and full) in all of its group, 0 for a sequence that shares none; a sequence that is in no group gets zeros.  ``shared_bound``, ``own_bound``: about how many pages a group
    shares and a sequence has of its own at most (for the caller's choice between this and ``decode``, see ``sharing_pays``; the kernel goes by the numbers themselves).  At most 1,024 sequences, and 1,024 tiles: of up to 16, 32 or 64 rows (members times heads of a kv head; the least that takes
    ``max_members``, else 64), counted as if every group had ``max_members`` (128 members of 4 heads: 8 tiles, so 128 such groups).  All else as ``decode`` has it, without a window."""
    n_pages, nkv, page_size, hd = k_pages.shape
    B, bf16, i32 = kv_lens.shape[0], torch.bfloat16, torch.int32
    if not supported(hd) or page_size != 64 or v_pages.shape != k_pages.shape:
        raise KernelError("decode_shared: pages of 64 keys and values of one head size, a multiple of 16 up to 256, are supported")
    if n_heads % nkv or q.numel() != B * n_heads * hd:
        raise KernelError(f"decode_shared: queries {tuple(q.shape)} are not {B} times {n_heads} heads of {hd} on {nkv} kv heads")
    dev = q.get_device()                           # -1 on the host
    if dev < 0 or dev != ops._current_device():
        ops._need(q, "q", bf16)
        ops._here(q, "q")
    for t, name, dtype in ((q, "q", bf16), (k_pages, "k_pages", bf16), (v_pages, "v_pages", bf16), (kv_lens, "kv_lens", i32), (starts, "starts", i32), (shared, "shared", i32)):
        if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
            ops._need(t, name, dtype)
            ops._here(t, name)
    if table.dtype is not i32 or table.get_device() != dev:
        ops._need(table, "table", i32, contiguous=False)
        ops._here(table, "table")
    sink_v = None if sink is False else ops.sink_values(sink, n_heads)
    for t, name in ((status, "status"), (sink_v, "the sink")):       # (handed to the kernel as addresses, like the rest)
        if t is not None and (t.get_device() != dev or t is status and t.dtype is not i32):
            ops._need(t, name, i32 if t is status else torch.float32)
            ops._here(t, name)
    if starts.numel() != n_groups + 1 or shared.numel() != B:
        raise KernelError(f"decode_shared: {n_groups + 1} starts and {B} numbers of shared pages are needed, found {starts.numel()} and {shared.numel()}")
    if shared_bound < 0 or own_bound < 0:
        raise KernelError("decode_shared: the bounds of the pages cannot be negative")
    if table.dim() != 2 or table.shape[0] != B or table.stride(1) != 1 or n_groups < 1 or not 1 <= max_members <= B:
        raise KernelError("decode_shared: the block table is [sequences, pages], and a group has between one and all of the sequences")
    m = shared_module(hd)
    key = (dev, hd, n_groups, max_members, B, n_heads, nkv)
    need = _shared_scratch.get(key)
    if need is None:
        if len(_shared_scratch) > 4096:
            _shared_scratch.clear()
        need = _shared_scratch[key] = m.ik_attn_shared_scratch(n_groups, max_members, B, n_heads, nkv)
    if need < 0:
        raise KernelError(f"decode_shared: {B} sequences in {n_groups} groups of up to {max_members} are more than this kernel takes")
    scratch = q.new_empty((need + 1) // 2)
    if out is None:
        out = torch.empty_like(q)
    else:
        ops._need(out, "out", bf16)
        ops._here(out, "out")
        if out.numel() != q.numel():
            raise KernelError(f"decode_shared: out has {out.numel()} elements, {q.numel()} are needed")
    if ops.profiling():
        ops._work(f"attention decode shared {B}x{n_heads}", *(work or (0, 0)))
    _check(m.ik_attn_shared(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), scratch.data_ptr(), kv_lens.data_ptr(), table.data_ptr(), table.stride(0),
                            table.shape[1], starts.data_ptr(), shared.data_ptr(), n_groups, max_members, B, n_heads, nkv, scale, softcap, ops.sink_flag(sink),
                            _ptr(sink_v), page_size, n_pages, _ptr(status), _stream()), "attention decode (shared pages)", kernels=2)
    return out


def attend(q, k_pages, v_pages, ctx, table, n_heads: int, scale: float, window: int,
           status, softcap: float = 0.0, sink=False, keep: int = 0,
            key_scales: Optional[torch.Tensor] = None, slopes: Optional[torch.Tensor] = None, reach=None, sharing=None) -> Optional[torch.Tensor]:
    """Returns None when no specialised kernel takes these sizes or options (the caller then uses the
    CUDA-core kernel).  ``sharing``: which neighbours of a decode step share their first pages (``engine.context.Sharing``), or None."""
    n_pages, nkv, page_size, hd = k_pages.shape
    if k_pages.dtype != torch.bfloat16 or q.dtype != torch.bfloat16 or page_size != 64 or not supported(hd):
        return None
    work = None
    if ops.profiling():
        # (query, key) pairs under the causal mask (and the window), from the host's copy of the lengths
        pairs = 0
        for n, end in zip(ctx.host_n_new, ctx.host_kv_lens):
            for p in range(end - n, end):
                pairs += min(p + 1, window + keep) if window else p + 1
        keys = sum(min(e, window + keep + n) if window else e for n, e in zip(ctx.host_n_new, ctx.host_kv_lens))
        rows = hd * 2 + 4 if key_scales is not None else 2 * hd * 2             # bytes of a key (and value) per kv head
        work = (2 * q.numel() * 2 + keys * nkv * rows, 4 * hd * n_heads * pairs)
    if (ctx.is_decode and sharing is not None and not window and key_scales is None and slopes is None
            and sharing_pays(ctx.n_seqs, sharing.n_groups, sharing.max_members, sharing.shared_bound, sharing.own_bound, n_heads, nkv, hd)):
        if work is not None:
            once = sum((b - a - 1) * sharing.pages[a] * page_size for a, b in zip(sharing.starts, sharing.starts[1:]))
            work = (work[0] - once * nkv * 4 * hd, work[1])
        return decode_shared(q, k_pages, v_pages, ctx.kv_lens, table, sharing.starts_dev, sharing.pages_dev, sharing.n_groups, sharing.max_members, sharing.shared_bound,
                             sharing.own_bound, n_heads, scale, status, softcap=softcap, sink=sink, work=work)
    if ctx.is_decode:
        # from the bound; the single lengths have a say only where the step is not captured: a graph is replayed for other lengths
        chunk = decode_chunk_pages(ctx.n_seqs, n_heads, nkv, seen_pages(ctx.kv_len_bound, window, keep, page_size) * page_size, page_size)
        if len(ctx.host_kv_lens) == ctx.n_seqs > 1 and not getattr(ctx, "replayed", False):
            key = ("decode_chunk", n_heads, nkv, window, keep, page_size)              # once for all layers of a kind
            if key not in ctx.shared:
                ctx.shared[key] = decode_chunk_pages_uneven([seen_pages(e, window, keep, page_size) for e in ctx.host_kv_lens], n_heads, nkv, chunk, sm_count())
            chunk = ctx.shared[key]
        options = {}
        if key_scales is not None or slopes is not None:
            options["ring_kb"] = OPTION_RING_KB
        if reach is not None:
            chunk = min(chunk, REACH_CHUNK_PAGES)
        return decode(q, k_pages, v_pages, ctx.kv_lens, table, ctx.n_seqs, ctx.kv_len_bound, n_heads, scale, window,
                      status, chunk_pages=chunk, work=work, **options, softcap=softcap, sink=sink, keep=keep, key_scales=key_scales, slopes=slopes, reach=reach)
    plain = hd in (64, 128) and key_scales is None and slopes is None and not softcap and not ops.sink_flag(sink) and not keep and n_heads // nkv % 2 == 0
    return prefill(q, k_pages, v_pages, ctx.cu_seqlens, ctx.kv_lens, table, ctx.n_seqs, ctx.max_new, n_heads, scale,
                   window, status, work=work, softcap=softcap, sink=sink, keep=keep, key_scales=key_scales, slopes=slopes, reach=reach,
                   two_heads=plain and _two_heads_of(ctx, n_heads, hd, int(window or 0)))
