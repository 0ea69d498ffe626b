"""Work items of the attention over lists of pages (``fk_paged_kv_attention``): how many pieces the tokens
of a group of query vectors are cut into, and the int32 rows that the kernel reads."""

from __future__ import annotations

import numpy as np

ITEM_ROWS = 256   # query rows (vectors x query heads of a kv head) of one item: FK_PAGED_KV_ITEM_ROWS
TILE_TOKENS = 128  # tokens that the kernel takes at a time
_SMS = 148
_ITEM_OVERHEAD = 4  # what an item costs besides its tiles, in tiles: queries in, results out, a pipeline to fill


def pieces_for(tiles: np.ndarray, kv_heads: int, fewest: int = 1) -> np.ndarray:
    """Pieces per group of vectors, `tiles[i]` tiles long, so that the items of all groups and kv heads fill
    the device evenly: the cut that is cheapest by waves of items times their mean length."""
    if tiles.size == 0:
        return np.zeros(0, dtype=np.int64)
    longest = int(tiles.max())
    most = -(-longest // np.arange(1, 65))  # tiles of a piece at most, for 1, 2, ... pieces of the longest
    most = most[: max(1, int((most >= fewest).sum()))][:, None]
    pieces = -(-tiles // most)
    size = -(-tiles // pieces)
    total = pieces.sum(axis=1)
    mean = (pieces * size).sum(axis=1) / total + _ITEM_OVERHEAD + (pieces.max(axis=1) > 1)  # (partial results are added up)
    costs = np.maximum(size.max(axis=1) + _ITEM_OVERHEAD, -(-(total * kv_heads) // _SMS) * mean).tolist()
    chosen = 0
    for index, cost in enumerate(costs):
        if cost < 0.97 * costs[chosen]:
            chosen = index
    return pieces[chosen]


def cut(first: np.ndarray, end: np.ndarray, pieces: np.ndarray) -> tuple[np.ndarray, np.ndarray, np.ndarray, np.ndarray]:
    """(group, number of the piece, first token, end token) of every piece of the token ranges [first, end); pieces begin
    a multiple of TILE_TOKENS behind `first` and none is empty unless its range is."""
    tiles = np.maximum(1, -(-(end - first) // TILE_TOKENS))
    size = -(-tiles // pieces)
    pieces = -(-tiles // size)
    group = np.repeat(np.arange(len(first)), pieces)
    number = np.arange(int(pieces.sum())) - np.repeat(np.cumsum(pieces) - pieces, pieces)
    begin = first[group] + number * size[group] * TILE_TOKENS
    return group, number, begin, np.minimum(begin + size[group] * TILE_TOKENS, end[group])


def item_rows(*, first_vector: np.ndarray, vectors: np.ndarray, entry: np.ndarray, first: np.ndarray, end: np.ndarray,
              causal: int, partial: np.ndarray, kv_heads: int) -> np.ndarray:
    """int32 [items * kv_heads, 8], the longest items first (the device takes them in order)."""
    order = np.argsort(-(-(-(end - first) // TILE_TOKENS)), kind="stable")
    rows = np.stack((first_vector, vectors, np.zeros_like(entry), entry, first, end, np.full_like(entry, causal), partial), axis=1)[order]
    rows = np.repeat(rows, kv_heads, axis=0)
    rows[:, 2] = np.tile(np.arange(kv_heads), len(order))
    return rows.astype(np.int32)
