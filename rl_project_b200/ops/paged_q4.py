"""Paged KV cache held in 4 bits (csrc/paged_q4.cu): storing and reading rows, decode attention, eviction.

Pools are uint8 ``[num_blocks, Hkv, q4_block_bytes(D)]`` for keys and for values, addressed like the bf16 pools of
``ops/paged_attention.py`` (16-token blocks, int32 block tables and context lengths).  Every group of
``min(D, 64)`` dimensions of a token's key or value keeps a bf16 minimum and scale and 4-bit codes::

    minimum = min x      scale = bf16((max x - min x) / 15)      code = clamp(rint((x - minimum) / scale), 0, 15)

and reads back as ``minimum + scale * code``; a group holding NaN or infinity reads back as NaN.  A token takes
``D / 2 + 4 D / min(D, 64)`` bytes, 0.28 of its bf16 size for D of 64 and 128.  Heads are 32, 64 or 128 wide.

Indexes are checked on the device: rows whose block, slot or accumulator row lies outside its table are skipped and
reported in ``status`` (int32, one element) or, without one, in the device's shared word that
``ops._ext.check_bounds`` reads.  On CPU tensors every operator runs its plain-PyTorch reference, which raises
``IndexError`` instead.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from rl_project_b200.ops._ext import native

BLOCK = 16
HEAD_DIMS = (32, 64, 128)


def q4_block_bytes(head_dim: int) -> int:
    """Bytes of one block (16 tokens of one KV head) of a 4-bit pool."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"the 4-bit cache has heads of 32, 64 or 128, got {head_dim}")
    return BLOCK * (head_dim // 2 + 4 * (head_dim // min(head_dim, 64)))


def paged_write_q4(k_new: torch.Tensor, v_new: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor,
                   slot_block: torch.Tensor, slot_off: torch.Tensor, status: Optional[torch.Tensor] = None) -> None:
    """Quantise row ``i`` of ``k_new / v_new [N, Hkv, D]`` (bf16, any strides) into block ``slot_block[i]``, slot
    ``slot_off[i]``.  The slots of one call must differ, unless their rows are equal."""
    if k_pool.is_cuda:
        native().q4_write(k_new, v_new, k_pool, v_pool, slot_block, slot_off, status)
        return
    _check_pools(k_pool, v_pool, k_new.shape[-1])
    if k_new.dim() != 3 or v_new.shape != k_new.shape or k_new.shape[1] != k_pool.shape[1]:
        raise ValueError("k_new, v_new: [N, Hkv, D]")
    _check_ints(slot_block, (k_new.shape[0],), "slot_block")
    _check_ints(slot_off, (k_new.shape[0],), "slot_off")
    blk, off = _slots(k_pool, slot_block, slot_off)
    for pool, x in ((k_pool, k_new), (v_pool, v_new)):
        codes, meta = _views(pool, k_new.shape[-1])
        c, m = _quantise(x.to(torch.bfloat16))
        codes[blk, :, off] = c
        meta[blk, :, off] = m


def paged_read_q4(k_pool: torch.Tensor, v_pool: torch.Tensor, slot_block: torch.Tensor, slot_off: torch.Tensor,
                  head_dim: int, status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values ``[N, Hkv, D]`` (bf16) stored in slots ``(slot_block[i], slot_off[i])``; slots outside
    the pool read as zeros."""
    if k_pool.is_cuda:
        k, v = native().q4_read(k_pool, v_pool, slot_block, slot_off, int(head_dim), status)
        return k, v
    _check_pools(k_pool, v_pool, head_dim)
    _check_ints(slot_block, (slot_block.numel(),), "slot_block")
    _check_ints(slot_off, (slot_block.numel(),), "slot_off")
    blk, off = _slots(k_pool, slot_block, slot_off)
    return tuple(_values(p, head_dim)[blk, :, off].to(torch.bfloat16) for p in (k_pool, v_pool))


def paged_gather_q4(k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                    head_dim: int, max_len: int,
                    status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first ``max_len`` keys and values of every sequence as ``[B, max_len, Hkv, D]`` (bf16), zeros behind a
    sequence's length."""
    if k_pool.is_cuda:
        k, v = native().q4_gather(k_pool, v_pool, block_tables, ctx_lens, int(head_dim), int(max_len), status)
        return k, v
    _check_pools(k_pool, v_pool, head_dim)
    _check_tables(block_tables, ctx_lens)
    out = [torch.zeros(ctx_lens.numel(), max_len, k_pool.shape[1], head_dim, dtype=torch.bfloat16) for _ in range(2)]
    for pool, to in zip((k_pool, v_pool), out):
        for b in range(ctx_lens.numel()):
            n = min(max_len, max(0, int(ctx_lens[b])))
            to[b, :n] = _sequence(pool, block_tables[b], n, head_dim).to(torch.bfloat16)
    return tuple(out)


def paged_decode_q4(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor,
                    ctx_lens: torch.Tensor, scale: float, softcap: float = 0.0, window: int = 0,
                    weights: Optional[torch.Tensor] = None, weight_rows: Optional[torch.Tensor] = None,
                    status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One query token per sequence over the 4-bit cache: ``q [B, Hq, D]`` bf16 -> ``[B, Hq, D]`` bf16, with up to 16
    query heads per KV head; a sequence of length 0 gives zeros.

    ``weights [rows, Hkv, tokens]`` (fp32) with ``weight_rows [B]`` (int32) accumulates, in row ``weight_rows[b]``,
    each cached token's attention weight summed over the query heads of its KV head (what ``paged_evict_q4`` ranks
    tokens by); a negative row accumulates nothing.  The rows of one call must differ.
    """
    if k_pool.is_cuda:
        return native().q4_decode(q, k_pool, v_pool, block_tables, ctx_lens, float(scale), float(softcap), int(window),
                                  weights, weight_rows, status)
    B, Hq, D = q.shape
    Hkv = k_pool.shape[1]
    _check_pools(k_pool, v_pool, D)
    _check_tables(block_tables, ctx_lens)
    if Hq % Hkv or Hq // Hkv > 16:
        raise ValueError("q: a multiple of the KV heads, at most 16 per KV head")
    if ctx_lens.numel() != B:
        raise ValueError("ctx_lens: one length per sequence")
    if (weights is None) != (weight_rows is None):
        raise ValueError("weights and weight_rows come together")
    if weights is not None:
        _check_weights(weights, weight_rows, k_pool, B)
    out = torch.zeros(B, Hq, D)
    for b in range(B):
        n = int(ctx_lens[b])
        if n <= 0:
            continue
        k, v = (_sequence(p, block_tables[b], n, D).transpose(0, 1) for p in (k_pool, v_pool))
        s = torch.einsum("hgd,htd->hgt", q[b].float().view(Hkv, -1, D), k) * scale
        if softcap > 0:
            s = torch.tanh(s / softcap) * softcap
        if 0 < window < n:
            s[..., :n - window] = float("-inf")
        p = s.softmax(-1)
        out[b] = torch.einsum("hgt,htd->hgd", p, v).reshape(Hq, D)
        if weights is not None and int(weight_rows[b]) >= 0:
            _inside(int(weight_rows[b]), weights.shape[0], "weight_rows")
            _inside(n - 1, weights.shape[2], "a context's last token")
            weights[int(weight_rows[b]), :, :n] += p.sum(1)
    return out.to(q.dtype)


def paged_evict_q4(k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                   new_tables: torch.Tensor, weights: torch.Tensor, weight_rows: torch.Tensor, keep: int, head_dim: int,
                   recent: int = 0, sink: int = 0,
                   status: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cut every sequence to at most ``keep`` cached tokens, separately for each KV head.

    The first ``sink`` and the last ``recent`` tokens stay; the other places go to the tokens with the largest
    accumulated ``weights`` (``paged_decode_q4``), the earliest among equals (NaN ranks lowest).  Kept tokens stay in
    order: their rows are copied to the blocks of ``new_tables [B, blocks]``, which must not be among the sequences'
    own blocks (those stay as they are, so they may be shared with other sequences), and their weights move to the
    front of their row (one to a sequence), the rest of the old length becoming zero.  A sequence of at most ``keep`` tokens is copied
    whole.  Returns ``(kept [B, Hkv, keep], new_lens [B])``, int32: the old positions (-1 behind the last) and lengths.
    """
    if k_pool.is_cuda:
        kept, lens = native().q4_evict(k_pool, v_pool, block_tables, ctx_lens, new_tables, weights, weight_rows,
                                       int(keep), int(head_dim), int(recent), int(sink), status)
        return kept, lens
    _check_pools(k_pool, v_pool, head_dim)
    _check_tables(block_tables, ctx_lens)
    _check_tables(new_tables, ctx_lens)
    B, Hkv = ctx_lens.numel(), k_pool.shape[1]
    _check_weights(weights, weight_rows, k_pool, B)
    if keep < 1 or recent < 0 or sink < 0 or recent + sink > keep:
        raise ValueError("keep at least one token, and no fewer than sink + recent")
    if new_tables.shape[1] * BLOCK < keep:
        raise ValueError("new_tables: blocks for `keep` tokens")
    kept = torch.full((B, Hkv, keep), -1, dtype=torch.int32)
    lens = ctx_lens.clamp(0, keep)
    for b in range(B):
        n, m = int(ctx_lens[b]), int(lens[b])
        if n <= 0:
            continue
        row = weights[_inside(int(weight_rows[b]), weights.shape[0], "weight_rows")]
        if n > keep:
            w = row[:, :n].nan_to_num(nan=float("-inf")).double()
            pos = torch.arange(n)
            w[:, (pos < sink) | (pos >= n - recent)] = float("inf")
            order = torch.sort(w, dim=1, descending=True, stable=True).indices[:, :keep].sort(1).values
            moved = row[:, :n].gather(1, order)
            row[:, :n] = 0
            row[:, :m] = moved
        else:
            order = torch.arange(n).expand(Hkv, n)
        kept[b, :, :m] = order.int()
        new = [_inside(int(new_tables[b, j]), k_pool.shape[0], "new_tables") for j in range(-(-m // BLOCK))]
        to = torch.tensor(new)[torch.arange(m) // BLOCK]
        old = torch.tensor([_inside(int(x), k_pool.shape[0], "block_tables") for x in block_tables[b, :-(-n // BLOCK)]])
        for pool in (k_pool, v_pool):
            for part in _views(pool, head_dim):
                for h in range(Hkv):
                    part[to, h, torch.arange(m) % BLOCK] = part[old[order[h] // BLOCK], h, order[h] % BLOCK]
    return kept, lens


# ------------------------------------------------------------------ plain reference of the layout
def _check_pools(k_pool, v_pool, head_dim: int) -> None:
    want = q4_block_bytes(head_dim)
    for p in (k_pool, v_pool):
        if p.dtype != torch.uint8 or p.dim() != 3 or p.shape[2] != want or not p.is_contiguous():
            raise ValueError(f"pool: contiguous uint8 [blocks, Hkv, {want}] for heads of {head_dim}")
    if k_pool.shape != v_pool.shape:
        raise ValueError("k_pool and v_pool differ in shape")


def _check_ints(t, shape, name: str) -> None:
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: int32 of shape {tuple(shape)} expected, got {t.dtype} {tuple(t.shape)}")


def _check_tables(tables, lens) -> None:
    _check_ints(lens, (lens.numel(),), "ctx_lens")
    _check_ints(tables, (lens.numel(), tables.shape[-1]), "block_tables")


def _check_weights(weights, rows, k_pool, B: int) -> None:
    if weights.dtype != torch.float32 or weights.dim() != 3 or weights.shape[1] != k_pool.shape[1]:
        raise ValueError("weights: fp32 [rows, Hkv, tokens]")
    _check_ints(rows, (B,), "weight_rows")


def _inside(i: int, n: int, name: str) -> int:
    if not 0 <= i < n:
        raise IndexError(f"{name}: {i} is outside 0..{n - 1}")
    return i


def _slots(pool, block, off):
    blk, off = block.long(), off.long()
    if blk.numel() and (blk.min() < 0 or blk.max() >= pool.shape[0] or off.min() < 0 or off.max() >= BLOCK):
        raise IndexError("a slot lies outside the pool")
    return blk, off


def _views(pool, D: int):
    """Codes and (scale, minimum) bytes of a pool as views [blocks, Hkv, 16, groups, bytes]."""
    g, n = min(D, 64), BLOCK * D // 2
    codes = pool[..., :n].unflatten(-1, (D // g, BLOCK, g // 2)).transpose(2, 3)
    meta = pool[..., n:].unflatten(-1, (D // g, BLOCK, 4)).transpose(2, 3)
    return codes, meta


def _quantise(x):
    """bf16 rows [..., D] -> code bytes [..., groups, group / 2] and (scale, minimum) bytes [..., groups, 4]."""
    x = x.float().unflatten(-1, (-1, min(x.shape[-1], 64)))
    lo, hi = x.amin(-1), x.amax(-1)
    scale = ((hi - lo) / 15).to(torch.bfloat16)
    n = ((x - lo[..., None]) / scale.float()[..., None]).nan_to_num(0.0).round().clamp(0, 15).to(torch.uint8)
    meta = torch.stack((scale, lo.to(torch.bfloat16)), -1).view(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), meta


def _values(pool, D: int) -> torch.Tensor:
    """What a pool's blocks stand for: fp32 [blocks, Hkv, 16, D]."""
    codes, meta = _views(pool, D)
    m = meta.contiguous().view(torch.bfloat16).float()
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    return (n * m[..., :1] + m[..., 1:]).flatten(-2)


def _sequence(pool, table, n: int, D: int) -> torch.Tensor:
    """The first ``n`` stored rows of a sequence, fp32 [n, Hkv, D]."""
    need = -(-n // BLOCK)
    if need > table.numel():
        raise IndexError(f"a context of {n} tokens is longer than its block table")
    blocks = table[:need].long()
    if need and (blocks.min() < 0 or blocks.max() >= pool.shape[0]):
        raise IndexError("block_tables: a block lies outside the pool")
    return _values(pool[blocks], D).transpose(1, 2).flatten(0, 1)[:n]
