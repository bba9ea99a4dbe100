"""The work partition of the paged attention, restated from its rules: which pieces a call is cut into, where their partial results go, how
much workspace and how many workgroups that takes.  Plain integers; the kernels find the same by scans over the lengths."""
from __future__ import annotations

STAGE = 128


class Plan:
    """share: stages of a piece (None: nothing is cut); per sequence tiles, stages, n (pieces per tile) and first_slot; limits of the launch."""

    def __init__(self, lengths, counts, H: int, Hkv: int, Lq: int, head_dim: int, f8: bool, max_len: int, cus: int, workspace: bool = True):
        G, B = H // Hkv, len(lengths)
        rows = G * Lq
        nt = 1 if rows <= 16 or head_dim == 256 else 2
        self.staged = rows > 16 * nt
        rw = 1 if not self.staged else 2 if rows <= 64 and head_dim < 256 else 4
        self.tile_rows = 16 * nt * rw
        self.rt = -(-rows // self.tile_rows)
        self.slot_rows = min(rows, self.tile_rows)
        i = head_dim // 128
        limit, more = (((8, 4, 2), (8, 8, 4)), ((4, 3, 2), (6, 6, 8)))[self.staged]
        whole = limit[i] + more[i] * min(B * Hkv * self.rt, cus) // cus
        self.finer = cus * (4 if self.staged else 6)
        stage_bytes = 2 * STAGE * head_dim * (1 if f8 else 2)
        per = (2 if self.rt > 1 else 1) if self.staged or nt == 2 else 1 if stage_bytes >= 65536 else 2 if stage_bytes >= 32768 else 3
        self.target, self.wide = per * cus, max(per, 2) * cus
        self.wider = 3 * cus if not self.staged and head_dim == 64 else self.wide
        self.some, self.many, self.most = (16 if not self.staged and nt == 2 and head_dim > 64 else 4) * cus, 16 * cus, 64 * cus
        singles = cus // 2 if self.staged else 0x7fffffff

        # workspace
        self.head = (2 * B + 63) // 64 * 64
        top = -(-max_len // STAGE)
        self.slots = min(B * Hkv * self.rt * top, 2 * self.finer)
        self.ws_bytes = 0 if top <= whole else 4 * (self.head + self.slots * self.slot_rows * (head_dim + 2))
        if not workspace or not self.ws_bytes:
            whole = 0x7fffffff

        self.stages = [max(1, -(-max(0, min(n, max_len)) // STAGE)) for n in lengths]
        fresh = [Lq] * B if counts is None else [max(0, min(c, Lq)) for c in counts]
        self.tiles = [max(1, -(-f * G // self.tile_rows)) for f in fresh]
        self.total = Hkv * sum(s * t for s, t in zip(self.stages, self.tiles))
        self.cut = any(s > whole for s in self.stages)

        def share_of(target):
            return max((self.total - 1) // target + 1, 2 if self.total > singles else 1)

        def pieces(share):
            return [1 if share is None or s <= 2 else (s - 1) // share + 1 for s in self.stages]

        def count(share):
            return Hkv * sum(n * t for n, t in zip(pieces(share), self.tiles))

        self.share, self.way = None, "uncut"
        if self.cut:
            self.share, self.way = share_of(self.target), "one round"
            if count(self.share) > self.target:
                self.way = "target" if self.total <= self.some or self.total > self.most else "wide" if self.total <= self.many else "wider"
                round_ = {"target": self.target, "wide": self.wide, "wider": self.wider}[self.way]
                even = share_of(round_)
                for x in range(1 if round_ == self.target else 0, 4):
                    self.share = even + x * max(1, even >> 3)
                    if count(self.share) <= round_:
                        break
                else:
                    self.share, self.way = share_of(self.finer), "finer"
        self.n = pieces(self.share)
        self.pieces = count(self.share)
        self.first_slot, slot = [], 0
        for n, t in zip(self.n, self.tiles):
            self.first_slot.append(slot)
            slot += n * t * Hkv if n > 1 else 0
        self.used_slots = slot
        items = B * Hkv * self.rt + (self.finer if workspace and self.ws_bytes else 0)
        self.grid = -(-items // 8) * 8
        self.Hkv = Hkv

    def item_of(self, wg: int):
        """Piece of a workgroup (None: left over): each of the 8 XCDs takes a run of them."""
        per = (self.pieces + 7) // 8
        item = wg % 8 * per + wg // 8
        return item if wg // 8 < per and item < self.pieces else None

    def piece(self, item: int):
        """(sequence, head, row tile, piece, first stage, stage behind the last, slot) of an item."""
        for b, (n, t) in enumerate(zip(self.n, self.tiles)):
            mine = n * t * self.Hkv
            if item < mine:
                tile, hp = item % t, item // t
                p, head = hp % n, hp // n
                s = self.stages[b]
                return b, head, tile, p, s * p // n, s * (p + 1) // n, self.first_slot[b] + item if n > 1 else None
            item -= mine
        raise IndexError(item)

    def join_slot(self, b: int, head: int, tile: int, p: int):
        """Where the join looks for a piece."""
        return self.first_slot[b] + head * self.n[b] * self.tiles[b] + tile + p * self.tiles[b]
