"""Paged cache of keys and values in 8 bits (float8 e4m3) with a scale for each page of 16 tokens and key head (``csrc/paged_fp8.cu``).

``qkv_append`` is everything between a fused projection and the attention: norms of the query and key heads, rotation, append of keys and values to
the pages. ``kv_attend`` is the attention of the same new tokens over all that the pages hold, one token a sequence or many, causal, with or without a
sliding window; ``tree_attend`` that of single rows with masks of their own. ``inference.kv_cache.PagedKVCache`` with ``fmt="fp8"`` calls them. They serve:
on a GPU no gradient and no tangent passes through them.

The scale of a page and head is the smallest power of two 2^e, at least 2^-64, with |x| <= 448 * 2^e for every token in it, keys as they are in fp32 behind
their norm and rotation (a first prompt and a later portion store the same; keys that were rounded before, to bf16, are rounded twice). Later tokens can raise it;
the codes that are there are then rounded to the new scale, which changes nothing but their exponent unless they fall under 2^-6. Tokens that are taken
back (a draft that was not accepted) leave the scale that they raised. A value that is not finite makes a page of its head read as NaN until its first slot
is written again."""
from __future__ import annotations

import functools
import struct
from typing import NamedTuple, Optional

import torch

from .. import _native
from . import runtime as rt
from .functional import _dense_rows, _head_norm_rope, _ld, _on16, _weights16, check_rope

_native.register_cuda_sigs({"inv_fp8_append": [_native.vp], "inv_fp8_attend": [_native.vp], "inv_fp8_attend_floats": [_native.i32] * 9})

# What the entries are given: their own pointers; the pools, page table, rows, cu, start, status and stream; heads, key heads, dim, pages, rows and width of
# the table, sequences, tokens; their own sizes; a number.
_APPEND = struct.Struct("=9Q 10Q 8q 5q d").pack
_ATTEND = struct.Struct("=7Q 10Q 8q 6q d").pack

PAGE, MIN_EXP = 16, -64
_e4m3, _fp32, _bf16, _int32 = torch.float8_e4m3fn, torch.float32, torch.bfloat16, torch.int32


class Fp8Pages(NamedTuple):
    """The pools of one layer, contiguous. Scales are powers of two from 2^-64 to 2^120, NaN in a page that holds no number, 0 in one never written."""
    k: torch.Tensor          # [pages, kv_heads, 16, dim] float8_e4m3fn
    v: torch.Tensor
    k_scale: torch.Tensor    # [pages, kv_heads] fp32
    v_scale: torch.Tensor


class NewTokens(NamedTuple):
    """Where a step's packed tokens belong: tokens [cu[i], cu[i + 1]) are the next ones of page table row ``rows[i]``, whose first ``start[i]`` positions
    are cached already. int32 on the pools' device; ``rows`` are distinct. Tokens in front of ``cu[0]`` and behind ``cu[n]`` are padding: what they would
    give stays as it is. The bounds size the launches, so a captured step is given the largest that it will be replayed with: no sequence has more than
    ``max_new`` tokens here, or ``max_len`` positions with them."""
    rows: torch.Tensor       # [n]
    cu: torch.Tensor         # [n + 1]
    start: torch.Tensor      # [n]
    max_new: int
    max_len: int


def new_pages(num_pages: int, kv_heads: int, dim: int, device) -> Fp8Pages:
    def codes():
        return torch.zeros(num_pages, kv_heads, PAGE, dim, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)

    def scales():
        return torch.zeros(num_pages, kv_heads, dtype=torch.float32, device=device)
    return Fp8Pages(codes(), codes(), scales(), scales())


def _check(x, what, heads, pages: Fp8Pages, page_table, kv_heads=None):
    """-> pages, key heads, size of a head. Asked in one expression, a few microseconds; what is wrong with arguments that fail is found by ``_refuse``."""
    k, v, ks, vs = pages
    shape, dev = k.shape, x.get_device()
    if (len(shape) == 4 and shape[2] == PAGE and shape[1] > 0 and v.shape == shape and k.dtype is _e4m3 and v.dtype is _e4m3
            and ks.shape == shape[:2] and vs.shape == shape[:2] and ks.dtype is _fp32 and vs.dtype is _fp32
            and k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()
            and heads > 0 and heads % shape[1] == 0 and (kv_heads is None or kv_heads == shape[1])
            and page_table.dim() == 2 and page_table.dtype is _int32 and page_table.is_contiguous() and page_table.numel() > 0
            and x.dim() == 2 and x.stride(1) == 1
            and dev == k.get_device() == v.get_device() == ks.get_device() == vs.get_device() == page_table.get_device()
            and (dev < 0 or (x.dtype is _bf16 and shape[3] in (64, 128)))):
        return shape[0], shape[1], shape[3]
    _refuse(x, what, heads, pages, page_table, kv_heads)


def _refuse(x, what, heads, pages, page_table, kv_heads):
    k = pages.k
    N, G, P, D = k.shape if k.dim() == 4 else (0, 0, 0, 0)
    if P != PAGE or pages.v.shape != k.shape or k.dtype != _e4m3 or pages.v.dtype != k.dtype:
        raise ValueError(f"pages of {k.dtype} {tuple(k.shape)} and {pages.v.dtype} {tuple(pages.v.shape)}: [pages, heads, {PAGE}, dim] of float8_e4m3fn")
    for s in (pages.k_scale, pages.v_scale):
        if s.shape != (N, G) or s.dtype != _fp32:
            raise ValueError(f"page scales of {s.dtype} {tuple(s.shape)}: fp32 {(N, G)}")
    if not all(t.is_contiguous() for t in pages):
        raise ValueError("pages and their scales are contiguous")
    if heads < 1 or G < 1 or heads % G or (kv_heads is not None and kv_heads != G):
        raise ValueError(f"{heads} query heads on pages of {G}")
    if page_table.dim() != 2 or page_table.dtype != _int32 or not page_table.is_contiguous() or page_table.numel() == 0:
        raise ValueError(f"page table of {page_table.dtype} {tuple(page_table.shape)}: contiguous int32 [rows, pages]")
    if x.dim() != 2 or x.stride(1) != 1:
        raise ValueError(f"{what} of {tuple(x.shape)}: rows of tokens with unit stride")
    if any(t.device != x.device for t in (*pages, page_table)):
        raise ValueError(f"{what} on {x.device}, pages on {k.device}, page table on {page_table.device}")
    if x.dtype != _bf16:
        raise TypeError(f"{what} in bf16 on a GPU, not {x.dtype}")
    raise ValueError(f"heads of {D}: 64 or 128 on a GPU")


def _check_new(new: NewTokens, x):
    rows, cu, start = new.rows, new.cu, new.start
    n, dev = rows.numel(), x.get_device()
    if not (cu.numel() == n + 1 and start.numel() == n and rows.dtype is _int32 and cu.dtype is _int32 and start.dtype is _int32
            and rows.is_contiguous() and cu.is_contiguous() and start.is_contiguous() and dev == rows.get_device() == cu.get_device() == start.get_device()):
        raise ValueError(f"rows, cu and start of {n} sequences: contiguous int32 on {x.device}")
    if n and (new.max_new < 1 or new.max_len < new.max_new):
        raise ValueError(f"max_new {new.max_new}, max_len {new.max_len}")
    return n


def _result(out, x, rows, width):
    """Where a call's result goes: new rows, or ``out``; with what the kernel writes, another tensor where ``out`` is not on 16-byte boundaries."""
    if out is None:
        out = torch.empty(rows, width, dtype=x.dtype, device=x.device)
        return out, out, width
    if out.shape != (rows, width) or out.dtype != x.dtype or out.device != x.device or out.stride(1) != 1:
        raise ValueError(f"out of {out.dtype} {tuple(out.shape)} for {rows} rows of {width}")
    if not x.is_cuda or _on16(out):
        return out, out, _ld(out)
    return out, out.clone(memory_format=torch.contiguous_format), width          # with its rows that the call leaves alone


def scale_of(amax: torch.Tensor) -> torch.Tensor:
    """The scale of pages with these largest values."""
    m, e = torch.frexp(amax.float())                           # amax = m 2^e, m in [1/2, 1); the largest code is 448 = 7/8 2^9
    e = torch.where(m == 0, MIN_EXP, torch.where(m > 0.875, e - 8, e - 9)).clamp(MIN_EXP, 120)
    return torch.where(torch.isfinite(amax), torch.ldexp(torch.ones_like(m), e), torch.nan)


def _write(x, codes, scales, page, slot):
    """x [tokens, kv_heads, dim] into slots [slot, slot + tokens) of one page, behind what is there."""
    new = scale_of(x.abs().amax((0, 2)))
    raw = codes.view(torch.uint8)
    if slot:
        old = scales[page].clone()
        new = torch.maximum(new, old)                          # NaN stays
        for h in torch.nonzero(new > old).flatten().tolist():
            raw[page, h, :slot] = (codes[page, h, :slot].float() * (old[h] / new[h])).to(codes.dtype).view(torch.uint8)
    y = (x.transpose(0, 1) / new.view(-1, 1, 1)).to(codes.dtype).view(torch.uint8)
    raw[page, :, slot:slot + x.shape[0]] = torch.where(torch.isnan(new).view(-1, 1, 1), torch.zeros_like(y), y)
    scales[page] = new


def _write_tokens(k, v, pages: Fp8Pages, ids, start: int):
    at, last = start, start + k.shape[0]
    while at < last:
        end = min(last, (at // PAGE + 1) * PAGE)
        for src, codes, scales in ((k, pages.k, pages.k_scale), (v, pages.v, pages.v_scale)):
            _write(src[at - start:end - start], codes, scales, ids[at // PAGE], at % PAGE)
        at = end


def _where(pages: Fp8Pages, page_table, rows, cu, start):
    k, v, ks, vs = pages
    return (k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), page_table.data_ptr(), rows, cu, start, rt.status_ptr(k), rt.stream_ptr())


def _places(new: NewTokens, page_table, pages: int, T: int, window: int = 0):
    """(first token, tokens, first position, page ids) of every sequence, on the CPU. What the table says of pages behind the window is not asked."""
    cu = new.cu.tolist()
    for i, (row, start) in enumerate(zip(new.rows.tolist(), new.start.tolist())):
        n = cu[i + 1] - cu[i]
        need = -(-(start + n) // PAGE)
        if not (0 <= cu[i] <= cu[i + 1] <= T and start >= 0 and 0 <= row < page_table.shape[0] and need <= page_table.shape[1] and n <= new.max_new):
            raise ValueError(f"sequence {i}: tokens [{cu[i]}, {cu[i + 1]}) of {T} at position {start} of row {row}")
        ids = page_table[row, :need].tolist()
        if window:
            behind = min(max(0, start - window + 1) // PAGE, need)
            ids[:behind] = [0] * behind
        if n and not all(0 <= p < pages for p in ids):
            raise ValueError(f"row {row} lists a page outside the pool of {pages}")
        yield cu[i], n, start, ids


def _check_weights(x, dim, *weights):
    for w in weights:
        if w is not None and (w.shape != (dim,) or w.dtype is not x.dtype or w.get_device() != x.get_device()):
            raise ValueError(f"head norm weight {w.dtype} {tuple(w.shape)} on {w.device} for {x.dtype} heads of {dim} on {x.device}")


def _check_positions(positions, x):
    if positions is not None and (positions.dtype != _int32 or positions.numel() != x.shape[0] or not positions.is_contiguous()
                                  or positions.device != x.device):
        raise ValueError(f"positions {positions.dtype} {tuple(positions.shape)}: contiguous int32, one for each of {x.shape[0]} tokens")


def _angles(cos, sin, positions, t0: int, m: int, start: int):
    """Cosines and sines [m, 1, pairs] of tokens [t0, t0 + m), on the CPU."""
    if cos is None:
        return None, None
    pos = torch.arange(start, start + m) if positions is None else positions[t0:t0 + m].long()
    if not (0 <= int(pos.min()) and int(pos.max()) < cos.shape[0]):
        raise ValueError(f"a position outside the tables of {cos.shape[0]}")
    return cos[pos].unsqueeze(1), sin[pos].unsqueeze(1)


def qkv_append(qkv, heads: int, kv_heads: int, dim: int, pages: Fp8Pages, page_table, new: NewTokens, cos=None, sin=None, positions=None, q_weight=None,
               k_weight=None, eps: float = 1e-6, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """qkv [T, (heads + 2 kv_heads) * dim]: packed tokens from the fused projection, bias included. Query and key heads are normed (``q_weight`` and
    ``k_weight`` [dim], or neither) and rotated (tables ``cos`` and ``sin`` [positions, pairs], of the first 2 * pairs values of a head, or neither) in
    fp32; keys and values go to the pages, whose other slots stay as they are. ``positions`` [T] int32: the rotation's, where they are not the
    tokens' places in their sequences. Returns the queries [T, heads * dim]. On a GPU an entry that points outside the tables or the pool is reported
    (``check_status`` raises) and its keys and values are not written."""
    N, G, D = _check(qkv, "qkv", heads, pages, page_table, kv_heads)
    T, width = qkv.shape
    if D != dim or width != (heads + 2 * G) * D:
        raise ValueError(f"qkv of {tuple(qkv.shape)} for {heads} query and {kv_heads} key heads of {dim} on pages of {D}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("norm weights of queries and keys, both or neither")
    _check_weights(qkv, D, q_weight, k_weight)
    rot = check_rope(cos, sin, D, qkv.device)
    n = _check_new(new, qkv)
    _check_positions(positions, qkv)
    q_out, to, ld_q = _result(q_out, qkv, T, heads * D)
    if not qkv.is_cuda:
        x = qkv.float().view(T, heads + 2 * G, D)
        for t0, m, start, ids in _places(new, page_table, N, T):
            if not m:
                continue
            c, s = _angles(cos, sin, positions, t0, m, start)
            part = x[t0:t0 + m]
            q_out[t0:t0 + m] = _head_norm_rope(part[:, :heads], q_weight, eps, c, s).reshape(m, -1).to(qkv.dtype)
            k, v = _head_norm_rope(part[:, heads:heads + G], k_weight, eps, c, s), part[:, heads + G:]
            _write_tokens(k, v, pages, ids, start)
        return q_out
    if rot % 16:
        raise ValueError(f"{rot} rotated values: a multiple of 16 on a GPU")
    if T == 0 or n == 0:
        return q_out
    qkv, ld = _dense_rows(qkv, width)
    q_weight, k_weight, cos, sin = _weights16(q_weight, k_weight, cos, sin)
    at, size = qkv.data_ptr(), D * qkv.element_size()
    with rt.device_of(qkv):
        rt.check(rt.lib().inv_fp8_append(_APPEND(at, at + heads * size, at + (heads + G) * size, to.data_ptr(), rt.ptr(q_weight), rt.ptr(k_weight),
                                                 rt.ptr(cos), rt.ptr(sin), rt.ptr(positions),
                                                 *_where(pages, page_table, new.rows.data_ptr(), new.cu.data_ptr(), new.start.data_ptr()),
                                                 heads, G, D, N, *page_table.shape, n, T, ld, ld, ld_q, cos.shape[0] if rot else 0, rot, eps)),
                 "inv_fp8_append")
    return q_out if to is q_out else q_out.copy_(to)


def kv_append(k, v, pages: Fp8Pages, page_table, new: NewTokens, cos=None, sin=None, positions=None, k_weight=None, eps: float = 1e-6):
    """Keys and values [T, kv_heads * dim] of packed tokens into the pages: ``qkv_append`` without queries, for those who norm and rotate them elsewhere.
    Key heads are normed with ``k_weight`` and rotated by the tables as there, and what is stored is the same to the bit; with neither they are stored as
    they are."""
    N, G, D = _check(k, "k", 1 if pages.k.dim() != 4 else pages.k.shape[1], pages, page_table)
    T = k.shape[0]
    if k.shape[1] != G * D or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device or v.stride(1) != 1:
        raise ValueError(f"k of {k.dtype} {tuple(k.shape)}, v of {v.dtype} {tuple(v.shape)} for {G} heads of {D}")
    _check_weights(k, D, k_weight)
    rot = check_rope(cos, sin, D, k.device)
    n = _check_new(new, k)
    _check_positions(positions, k)
    if not k.is_cuda:
        for t0, m, start, ids in _places(new, page_table, N, T):
            if m:
                c, s = _angles(cos, sin, positions, t0, m, start)
                keys = _head_norm_rope(k[t0:t0 + m].float().view(m, G, D), k_weight, eps, c, s)
                _write_tokens(keys, v[t0:t0 + m].float().view(m, G, D), pages, ids, start)
        return
    if rot % 16:
        raise ValueError(f"{rot} rotated values: a multiple of 16 on a GPU")
    if T == 0 or n == 0:
        return
    (k, ld), (v, ld_v) = _dense_rows(k, G * D), _dense_rows(v, G * D)
    k_weight, cos, sin = _weights16(k_weight, cos, sin)
    with rt.device_of(k):
        rt.check(rt.lib().inv_fp8_append(_APPEND(0, k.data_ptr(), v.data_ptr(), 0, 0, rt.ptr(k_weight), rt.ptr(cos), rt.ptr(sin), rt.ptr(positions),
                                                 *_where(pages, page_table, new.rows.data_ptr(), new.cu.data_ptr(), new.start.data_ptr()),
                                                 0, G, D, N, *page_table.shape, n, T, ld, ld_v, 0, cos.shape[0] if rot else 0, rot, eps)), "inv_fp8_append")


def read(pages: Fp8Pages, ids: torch.Tensor, length: int):
    """Keys and values [length, kv_heads, dim] in fp32 of a sequence in pages ``ids``."""
    out = []
    for codes, scales in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)):
        x = codes.view(torch.uint8)[ids.long()].view(codes.dtype).float() * scales[ids.long()][..., None, None]
        out.append(x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:length])
    return out[0], out[1]


def _softmax_rows(q, k, v, scale, seen):
    """q [rows, heads, dim], k and v [keys, kv_heads, dim], seen [rows, keys] -> [rows, heads * dim] fp32; a row that sees nothing gives zeros."""
    G = k.shape[1]
    s = torch.einsum("tghd,jgd->ghtj", q.float().view(q.shape[0], G, -1, q.shape[2]), k) * scale
    p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
    p = torch.where(seen.any(-1, keepdim=True), p, torch.zeros_like(p))
    o = torch.einsum("ghtj,jgd->tghd", p, torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0))
    lost = torch.einsum("tj,jgd->tgd", seen.float(), (~torch.isfinite(v)).float()) > 0        # a hidden value is nothing, whatever it holds
    return o.masked_fill(lost.unsqueeze(2), float("nan")).reshape(q.shape[0], -1)


@functools.lru_cache(maxsize=1024)
def _floats(n, T, heads, kv_heads, dim, max_new, max_len, window, tree):
    fn = rt.lib().inv_fp8_attend_floats
    fn.restype = _native.i64
    return fn(n, T, heads, kv_heads, dim, max_new, max_len, window, tree)


def _workspace(dev, *sizes):
    """Partial results of a split attention, and how many values. A call's own, so that calls on two streams and captured graphs share none."""
    floats = _floats(*sizes)
    return torch.empty(floats, dtype=torch.float32, device=dev) if floats else None, floats


def kv_attend(q, pages: Fp8Pages, page_table, new: NewTokens, heads: int, scale: Optional[float] = None, window: int = 0,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [T, heads * dim]: the queries of ``new``'s tokens, whose keys and values are in the pages already. The token at position p of its sequence
    sees the positions up to p, or with ``window`` > 0 the latest ``window`` of them, its own included; pages that all of a sequence's new tokens have
    left behind are not looked up. Query head h uses key head h // (heads / kv_heads). Returns [T, heads * dim]. On a GPU calls of many rows take scores
    (scale q.k) up to 5.8 million; where a row's largest is beyond that ``check_status`` raises."""
    N, G, D = _check(q, "q", heads, pages, page_table)
    T, width = q.shape
    if width != heads * D or window < 0:
        raise ValueError(f"q of {tuple(q.shape)} for {heads} heads of {D}, window {window}")
    n = _check_new(new, q)
    scale = D ** -0.5 if scale is None else float(scale)
    out, to, ld_o = _result(out, q, T, width)
    if not q.is_cuda:
        for t0, m, start, ids in _places(new, page_table, N, T, window):
            if m:
                k, v = read(pages, torch.tensor(ids), start + m)
                p, j = torch.arange(start, start + m).view(-1, 1), torch.arange(start + m)
                seen = (j <= p) & (j > p - window) if window else j <= p
                out[t0:t0 + m] = _softmax_rows(q[t0:t0 + m].view(m, heads, D), k, v, scale, seen).to(q.dtype)
        return out
    if T == 0 or n == 0:
        return out
    q, ld = _dense_rows(q, width)
    window = min(window, 2 ** 31 - 1)
    with rt.device_of(q):
        work, floats = _workspace(q.device, n, T, heads, G, D, new.max_new, new.max_len, window, 0)
        rt.check(rt.lib().inv_fp8_attend(_ATTEND(q.data_ptr(), to.data_ptr(), rt.ptr(work), 0, 0, 0, 0,
                                                 *_where(pages, page_table, new.rows.data_ptr(), new.cu.data_ptr(), new.start.data_ptr()),
                                                 heads, G, D, N, *page_table.shape, n, T, ld, ld_o, window, new.max_new, new.max_len, floats, scale)),
                 "inv_fp8_attend")
    return out if to is out else out.copy_(to)


def tree_attend(q, pages: Fp8Pages, page_table, seq_lens, row_seq, heads: int, max_len: int, scale: Optional[float] = None, tail_start=None,
                tail_mask=None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows with masks of their own: row t of q [T, heads * dim] belongs to page table row ``row_seq[t]``, which holds ``seq_lens[row_seq[t]]`` tokens,
    and sees those below ``tail_start[t]`` and token ``tail_start[t] + i``, i < 64, iff bit i of ``tail_mask[t]`` (int64) is set; all of them without a
    tail. A row that sees nothing gives zeros. No row of the page table holds more than ``max_len`` tokens. On a GPU a row outside the table, or one that
    would hold more than the table lists, gives zeros, a page outside the pool is skipped, and ``check_status`` raises."""
    N, G, D = _check(q, "q", heads, pages, page_table)
    T, width = q.shape
    if width != heads * D or max_len < 1 or (tail_start is None) != (tail_mask is None):
        raise ValueError(f"q of {tuple(q.shape)} for {heads} heads of {D}, max_len {max_len}, tail_start and tail_mask both or neither")
    for t, size, dt in ((seq_lens, page_table.shape[0], torch.int32), (row_seq, T, torch.int32), (tail_start, T, torch.int32), (tail_mask, T, torch.int64)):
        if t is not None and (t.dtype != dt or t.numel() != size or not t.is_contiguous() or t.device != q.device):
            raise ValueError(f"{tuple(t.shape)} {t.dtype} on {t.device}: contiguous {dt} [{size}] on {q.device}")
    scale = D ** -0.5 if scale is None else float(scale)
    out, to, ld_o = _result(out, q, T, width)
    if not q.is_cuda:
        lens, starts, masks = seq_lens.tolist(), tail_start.tolist() if tail_start is not None else None, tail_mask.tolist() if tail_mask is not None else None
        for t, row in enumerate(row_seq.tolist()):
            if not (0 <= row < page_table.shape[0] and 0 <= lens[row] <= PAGE * page_table.shape[1]):
                raise ValueError(f"row {t} of table row {row}" + (f", which holds {lens[row]} tokens" if 0 <= row < len(lens) else f" of {len(lens)}"))
            ids = page_table[row, : -(-lens[row] // PAGE)]
            if lens[row] and not (0 <= int(ids.min()) and int(ids.max()) < N):
                raise ValueError(f"row {row} lists a page outside the pool of {N}")
            k, v = read(pages, ids, lens[row])
            j = torch.arange(lens[row])
            seen = torch.ones(lens[row], dtype=torch.bool)
            if starts is not None:
                bits = torch.tensor([(masks[t] >> i) & 1 for i in range(64)] + [0], dtype=torch.bool)
                seen = (j < starts[t]) | bits[(j - starts[t]).clamp(0, 64)]
            out[t] = _softmax_rows(q[t].view(1, heads, D), k, v, scale, seen.view(1, -1))[0].to(q.dtype)
        return out
    if T == 0:
        return out
    q, ld = _dense_rows(q, width)
    with rt.device_of(q):
        work, floats = _workspace(q.device, T, T, heads, G, D, 1, max_len, 0, 1)
        rt.check(rt.lib().inv_fp8_attend(_ATTEND(q.data_ptr(), to.data_ptr(), rt.ptr(work), row_seq.data_ptr(), seq_lens.data_ptr(), rt.ptr(tail_start),
                                                 rt.ptr(tail_mask), *_where(pages, page_table, 0, 0, 0),
                                                 heads, G, D, N, *page_table.shape, T, T, ld, ld_o, 0, 1, max_len, floats, scale)), "inv_fp8_attend")
    return out if to is out else out.copy_(to)
