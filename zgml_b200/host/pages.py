"""Paged caches in 8 bits on the host (PAGE_APPEND, PAGED_ATTENTION, PAGE_READ, PAGE_COPY): which pages a sequence has, what has to be copied before a step writes, and
the bytes of a page."""
from typing import Dict, List, Sequence, Tuple

import numpy as np

from .. import abi

PAGE_TOKENS = (16, 32, 64)


def _padded(n: int, step: int) -> int:
    return -(-n // step) * step


def page_words(kv_heads: int, dk: int, dv: int, page_tokens: int) -> int:
    """f32 slots of a page of all key heads."""
    if page_tokens not in PAGE_TOKENS or kv_heads < 1 or not (0 < dk <= 256 and 0 < dv <= 256):
        raise ValueError(f"pages of {page_tokens} tokens of {kv_heads} heads of {dk} and {dv} values")
    return kv_heads * (16 + page_tokens * (_padded(dk, 32) + _padded(dv, 16))) // 4


def pack_pages(keys: np.ndarray, values: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """The words of pages (int32 [pages, page_words]) with codes keys [pages, heads, tokens, dk] and values [pages, heads, tokens, dv] (int8, -127 to 127) and scales [pages, heads, 2]
    (of keys and of values)."""
    P, G, tokens, dk = keys.shape
    dv = values.shape[3]
    page_words(G, dk, dv, tokens)
    if values.shape[:3] != (P, G, tokens) or scales.shape != (P, G, 2):
        raise ValueError("keys, values and scales of different pages")

    def padded(codes, step):
        c = np.full((P, G, tokens, _padded(codes.shape[3], step)), 128, np.uint8)
        c[..., :codes.shape[3]] = codes.astype(np.int16) + 128
        return c
    k = padded(keys, 32).reshape(P, G, tokens // 8, 8, -1, 32).swapaxes(3, 4)
    v = padded(values, 16).reshape(P, G, tokens // 16, 2, 4, 2, -1, 2, 8).transpose(0, 1, 2, 6, 8, 4, 7, 3, 5)
    head = np.zeros((P, G, 4), np.float32)
    head[..., :2] = scales
    return np.concatenate([head.view(np.uint8), k.reshape(P, G, -1), v.reshape(P, G, -1)], 2).reshape(P, -1).view(np.int32)


def unpack_pages(words: np.ndarray, kv_heads: int, dk: int, dv: int, page_tokens: int) -> Tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Codes and scales, as pack_pages takes them, of pages' words."""
    G, tokens, kp, vp = kv_heads, page_tokens, _padded(dk, 32), _padded(dv, 16)
    b = np.ascontiguousarray(words).view(np.uint8).reshape(-1, 4 * page_words(G, dk, dv, tokens) // G).reshape(-1, G, 16 + tokens * (kp + vp))
    P, codes = b.shape[0], (b[..., 16:].astype(np.int16) - 128).astype(np.int8)
    k = codes[..., :tokens * kp].reshape(P, G, tokens // 8, kp // 32, 8, 32).swapaxes(3, 4).reshape(P, G, tokens, kp)
    v = codes[..., tokens * kp:].reshape(P, G, tokens // 16, vp // 16, 8, 4, 2, 2, 2).transpose(0, 1, 2, 7, 5, 8, 3, 6, 4).reshape(P, G, tokens, vp)
    return k[..., :dk].copy(), v[..., :dv].copy(), np.ascontiguousarray(b[..., :8]).view(np.float32)


def move_words(moves: int) -> int:
    """f32 slots of the table of a PAGE_COPY of at most `moves` pages."""
    return abi.BATCH_ROWS + abi.BATCH_WORDS * moves


def page_moves(moves: Sequence[Tuple[int, int]], most: int, pages: int) -> np.ndarray:
    """The table of a PAGE_COPY of at most `most` pages in a pool of `pages`: (source, destination) pairs, which all run at once."""
    if len(moves) > most:
        raise ValueError(f"{len(moves)} moves for a copy of {most}")
    sources, to = {s for s, _ in moves}, [d for _, d in moves]
    if any(not 0 <= p < pages for m in moves for p in m):
        raise ValueError("a move outside the pool")
    if len(set(to)) < len(to) or sources & set(to):
        raise ValueError("a page that one move writes is written or read by another")
    t = np.zeros(move_words(most), np.int32)
    t[0] = len(moves)
    if moves:
        t[abi.BATCH_ROWS:].reshape(most, abi.BATCH_WORDS)[:len(moves), :2] = moves
    return t


class PagePool:
    """Which pages of a pool the slots' sequences have.  Sequences may share pages (fork); a page that several have is copied before one of them writes to it: `extend` and
    `compact` return the copies as (source, destination) pairs, which have to run (PAGE_COPY, once per pool that the pages stand for) before the step that uses `table`.  Lists of several calls
    run one after the other, or together, in one PAGE_COPY, if each call was given the copies of those before it that had not run (`pending`): `moves += pool.extend(slot, 1, moves)`."""

    def __init__(self, pages: int, page_tokens: int, slots: int, most: int):
        if page_tokens not in PAGE_TOKENS or pages < 1 or slots < 1 or most < 1:
            raise ValueError(f"a pool of {pages} pages of {page_tokens} tokens for {slots} slots of {most}")
        self.pages, self.page_tokens, self.most = pages, page_tokens, most
        self.table = np.zeros((slots, most), np.int32)
        self.lengths = [0] * slots
        self._held: List[List[int]] = [[] for _ in range(slots)]
        self._users = [0] * pages
        self._free = list(range(pages - 1, -1, -1))                  # the lowest first

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def page_ids(self, slot: int) -> List[int]:
        return list(self._held[slot])

    def _set(self, slot: int):
        held = self._held[slot]
        self.table[slot, :len(held)] = held
        self.table[slot, len(held):] = 0

    def _give_back(self, page: int):
        self._users[page] -= 1
        if not self._users[page]:
            self._free.append(page)
            self._free.sort(reverse=True)

    def extend(self, slot: int, tokens: int, pending: Sequence[Tuple[int, int]] = ()) -> List[Tuple[int, int]]:
        """Room for `tokens` more positions of the slot's sequence; returns the copies to make first.  Where the pool has no room, or no page for a copy that those in `pending` leave alone (when they
        have run there may be one), RuntimeError, and nothing has changed."""
        if tokens < 0:
            raise ValueError(f"{tokens} more positions")
        held, start, end = self._held[slot], self.lengths[slot], self.lengths[slot] + tokens
        if end > self.most * self.page_tokens:
            raise ValueError(f"slot {slot} would reach position {end}: its page table has {self.most} pages of {self.page_tokens}")
        if not tokens:
            return []
        first = start // self.page_tokens
        shared = [n for n in range(first, len(held)) if self._users[held[n]] > 1]
        new = max(0, -(-end // self.page_tokens) - len(held))
        if len(shared) + new > len(self._free):
            raise RuntimeError(f"no free page for slot {slot}: {len(shared) + new} wanted, {len(self._free)} free")
        touched, origin = {p for m in pending for p in m}, {d: s for s, d in pending}
        copied = [n for n in shared if n * self.page_tokens < start]      # (only the page that holds positions already needs its bytes)
        if copied and touched.issuperset(self._free):
            raise RuntimeError(f"no free page for slot {slot} that the copies before do not touch")
        moves = []
        for n in shared:
            if n in copied:
                page = next(p for p in reversed(self._free) if p not in touched)
                self._free.remove(page)
                moves.append((origin.get(held[n], held[n]), page))
            else:
                page = self._free.pop()
            self._users[held[n]] -= 1
            self._users[page], held[n] = 1, page
        for _ in range(new):
            page = self._free.pop()
            self._users[page] = 1
            held.append(page)
        self.lengths[slot] = end
        self._set(slot)
        return moves

    def fork(self, slot: int, to: int, length: int = None):
        """The free slot `to` begins as the first `length` positions (all) of slot's sequence, in the same pages: positions that steps have written, since a copy runs before its step."""
        length = self.lengths[slot] if length is None else length
        if slot == to or self._held[to] or not 0 <= length <= self.lengths[slot]:
            raise ValueError(f"{length} positions of slot {slot}, which has {self.lengths[slot]}, to slot {to}")
        self._held[to] = self._held[slot][:-(-length // self.page_tokens)]
        for page in self._held[to]:
            self._users[page] += 1
        self.lengths[to] = length
        self._set(to)

    def shrink(self, slot: int, length: int):
        """The slot's sequence ends at `length` (drafts that were not taken); pages behind it are given back."""
        if not 0 <= length <= self.lengths[slot]:
            raise ValueError(f"{length} positions of slot {slot}, which has {self.lengths[slot]}")
        keep = -(-length // self.page_tokens)
        for page in self._held[slot][keep:]:
            self._give_back(page)
        del self._held[slot][keep:]
        self.lengths[slot] = length
        self._set(slot)

    def release(self, slot: int):
        self.shrink(slot, 0)

    def compact(self, pending: Sequence[Tuple[int, int]] = ()) -> List[Tuple[int, int]]:
        """Moves the pages in use to the lowest numbers, those aside that copies in `pending` touch; returns the copies to make before the next step."""
        touched, origin = {p for m in pending for p in m}, {d: s for s, d in pending}
        live = [p for p in range(self.pages) if self._users[p]]
        holes = [p for p in range(len(live)) if not self._users[p] and p not in touched]
        to: Dict[int, int] = dict(zip([p for p in live if p >= len(live)], holes))
        for source, dst in to.items():
            self._users[dst], self._users[source] = self._users[source], 0
        for slot, held in enumerate(self._held):
            self._held[slot] = [to.get(p, p) for p in held]
            self._set(slot)
        self._free = [p for p in range(self.pages - 1, -1, -1) if not self._users[p]]
        return [(origin.get(source, source), dst) for source, dst in to.items()]
