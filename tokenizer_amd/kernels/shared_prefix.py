"""What the requests of a batch share: runs of leading pages that several block tables have in common, and the list of work
that the attention kernel makes of them (`csrc/attention_shared_prefix.hip`).  Host side, NumPy."""
from __future__ import annotations

import dataclasses

import numpy as np
import torch

WAVE = 64                         # lanes of a wave, which looks at so many parts at a time when they are joined


@dataclasses.dataclass
class SharedRun:
    """Keys `key_begin` .. `key_end` - 1 are the same for the `rows` (indices into the batch)."""
    rows: list[int]
    key_begin: int
    key_end: int


def find_shared_runs(block_table, positions, page_size: int, min_keys: int):
    """The runs of keys that at least two rows share, and where each row's own keys begin.

    block_table int [B, P], positions (of the rows' newest tokens) int [B].  Two rows share a page when their tables name it at the
    same place and everything before it too; only pages that are full for every row count, so a plan holds as long as the rows'
    positions do not fall.  Sharing may branch: all rows share a first part, some of them a further one.  A run of fewer than
    `min_keys` keys is not one of its own: the keys stay with the runs behind it, or with the rows.

    Returns (order, runs, own_begin): the rows so that those of any run stand side by side; the runs, those of shorter prefixes
    first; int32 [B]."""
    table = np.ascontiguousarray(block_table, dtype=np.int32)
    n_rows, width = table.shape
    full = np.minimum((np.asarray(positions, dtype=np.int64) + 1) // page_size, width).clip(min=0)
    # A page that is not full, or not there, is like no other row's.
    known = (np.arange(width)[None] < full[:, None]) & (table >= 0)
    full = np.where(known.all(axis=1), width, known.argmin(axis=1)) if width else full
    marked = np.where(np.arange(width)[None] < full[:, None], table, -1 - np.arange(n_rows, dtype=np.int32)[:, None])
    sortable = marked.astype(">u4")                       # (as unsigned bytes, the highest first: equal rows meet)
    order = sorted(range(n_rows), key=lambda row: sortable[row].tobytes())
    sorted_rows = marked[order]
    common = np.zeros(max(0, n_rows - 1), dtype=np.int64)           # pages that neighbours in the order have in common
    if n_rows > 1:
        differs = sorted_rows[1:] != sorted_rows[:-1]
        common = np.where(differs.any(axis=1), differs.argmax(axis=1), width)
    runs, own_pages = [], np.zeros(n_rows, dtype=np.int32)
    open_ranges = [(0, n_rows, 0)]
    while open_ranges:
        low, high, depth = open_ranges.pop()
        if high - low < 2:
            own_pages[order[low:high]] = depth
            continue
        shared = int(common[low:high - 1].min())
        if (shared - depth) * page_size >= min_keys:
            runs.append(SharedRun([int(r) for r in order[low:high]], depth * page_size, shared * page_size))
            depth = shared
        if shared == width:                               # (rows that are all alike)
            own_pages[order[low:high]] = depth
            continue
        starts = [low] + [low + 1 + int(i) for i in np.nonzero(common[low:high - 1] == shared)[0]] + [high]
        open_ranges += [(a, b, depth) for a, b in zip(starts, starts[1:])]
    runs.sort(key=lambda run: (run.key_begin, -len(run.rows)))
    return order, runs, own_pages * page_size


class SharedPrefixes:
    """A batch's sharing laid out for the attention kernel: made once (`Ops.plan_shared_prefixes`) for requests that stay the same,
    used at every layer and step.  It belongs to rows in this order with these leading pages, and to one shape of attention."""

    # Query columns (requests x query heads of a kv head) of an item: of few, whose waves share out the keys; of many, likewise; of many in
    # bfloat16 at head sizes WIDE_HEADS, whose waves have 32 each and keys and values come through LDS.
    FEW_COLUMNS, MANY_COLUMNS, WIDE_COLUMNS = 16, 32, 128
    WIDE_HEADS = (64, 128)
    # Items of many columns read the keys less often but are fewer, so they pay where the runs have so many scores (columns x keys x kv
    # heads, of all runs); below, every item is one of few.  Few only | with many, us: head size 128, 4 kv heads of 7 query heads,
    # 4,096 shared keys, 16 requests (1.8 million) 14 | 17, 24 15.4 | 18.8, 32 (3.7) 20.2 | 19.6, 100 44 | 30; 256 requests behind 32,000
    # 554 | 146.  Head size 64, 2 kv heads, 4,096 keys, 64 requests (3.7) 12.9 | 14.0, 100 16.0 | 15.6; 128 behind 2,048 in families
    # of 512 more (4.6) 20.7 | 14.9.  In 32 bits, 4,096 keys, 8 requests 12.1 | 17.4, 128 (7) 35.7 | 41.6; behind 16,000 64 (14) 54 | 63,
    # 128 (29) 104 | 87.  Head size 96, 4,096 keys, 256 requests (15) 30.0 | 27.2; behind 16,000 64 (14) 26 | 30, 256 (57) 87 | 56.
    WIDE_WORK, MANY_WORK = 3_700_000, 16_000_000
    # ... and what is left of a run's columns, up to so many, goes into items of few all the same.  (64 left, behind 4,096 keys, up to 64 | 48:
    # 28.1 | 24.7 us.)
    WIDE_LITTLE, MANY_LITTLE = 48, 16
    # A shorter run is not a pass and a part to be joined of its own.  (64 requests, 64 keys shared 14.7 us as a run, 14.0 with the
    # requests' own; 256 keys 19.2 and 19.2, and the cache is read less.)
    MIN_KEYS = 64
    # Keys of a part of a run, at least: a block of 32 for each of its four waves, four blocks of 64 where many columns go through LDS.  (Parts of
    # 64 | 128 | 256 keys, 2 requests of 4,096 keys 13.1 | 10.6 | 10.6 us, 4 requests of 512 7.4 | 7.1 | 7.8; 128 | 256 | 512 keys, many
    # columns, 64 requests of 4,096 29.7 | 24.7 | 25.4, of 1,024 17.4 | 17.4 | 21.5.)  Of a long run a 64th (a wave joins 64 parts at a time) or,
    # through LDS, a 16th, up to LONG_PART: 2 requests of 32,000 keys of head size 64 in 250 parts 25.8 us, in 63 12.8; 64 of 8,192 in parts
    # of 256 | 512 32.0 | 28.8.
    MIN_PART, MIN_WIDE_PART, LONG_PART = 128, 256, 512
    # The requests' own keys, in parts of one length, about so many of all requests together (as for single tokens that share nothing).  Each
    # request has as many as its own keys are planned to come to, in steps of OWN_STEP, so a long one among short ones has many, up to what a wave
    # joins at a time.  (Requests behind 4,096 keys, 256 behind 8,192, with 100 to 300 of their own, and one of 32,000 that shares nothing: 256 of
    # 28 query heads of size 128, as many parts for each as for the longest 403 us, so 87; 64 of them 149 | 42; 64 of 14 heads of size 64 48 | 20;
    # 8 of those 22 | 15, in 257 parts 28.)
    OWN_TARGET, OWN_STEP = 1024, 512
    # Workgroups that the parts aim at: two a compute unit; one where all items are of few columns.  (256 | 512 | 768: 64 requests behind 4,096
    # keys 34.6 | 28.7 | 32.7 us, 256 behind 32,000 187 | 145 | 161; few only, 64 behind 512 11.0 | 13.1 | 13.2, 24 behind 4,096
    # 15.5 | 18.5 | 18.2, 16 15.1 | 14.2 | 18.1, 2 behind 32,000 22.0 | 26.7 | 32.7.)
    TARGET, FEW_TARGET = 512, 256

    # Whether going through shared keys once is faster than each request's going through them by itself (`pays`): it spares the reading of so many
    # bytes of keys and values, and costs a launch that joins the parts where the other way often has none; in bfloat16 that one has none for
    # contexts of up to WHOLE_KEYS and from WHOLE_ROWS rows x kv heads on.  (Each alone | shared, us in captured steps, 40 keys of their own: 14 query
    # heads of size 64, 2 kv heads, bfloat16, 2 requests of 256 keys 5.1 | 7.1, of 4,096 7.5 | 10.1; 8 of 4,096 (14.7 MB) 9.7 | 10.3, 16 of
    # 4,096 (31) 10.5 | 10.1; 64 of 512 (16.5) 8.8 | 8.3, of 4,096 18.0 | 12.7; 128 of 512 6.8 | 9.2, of 1,024 12.9 | 10.5.  28 heads of 128,
    # 4 kv heads, 8 of 1,024 (14.7) 9.6 | 10.0, 4 of 4,096 (25) 14.7 | 12.1, 64 of 4,096 57 | 20.  In 32 bits, 14 heads of 64, 4 of 2,048 (6.3)
    # 9.8 | 10.6, 8 of 2,048 (14.7) 11.4 | 10.6, 64 of 2,048 26.1 | 15.7.  Over 732 such pairs of three more shapes, and with 400 keys of their own, this
    # rule is 0.8 % off the faster one on average, always sharing 12.8 %.  At worst, 32 of 256 keys of size 128 in 32 bits, 15.4 for 11.1.)
    PAYS_FROM, WHOLE_KEYS, WHOLE_ROWS = 16_000_000, 1024, 128

    def __init__(self, block_table, positions, page_size: int, n_q: int, n_kv: int, head_dim: int, dtype: torch.dtype, device,
                 fill: bool = False, growth: int | None = None):
        table = np.asarray(block_table, dtype=np.int32)
        self.n_rows, self.page_size, self.n_q, self.n_kv, self.head_dim, self.dtype = (
            table.shape[0], int(page_size), int(n_q), int(n_kv), int(head_dim), dtype)
        self.belongs_to = (self.n_rows, self.n_q, self.n_kv, self.head_dim, dtype)
        self.order, self.runs, own_begin = find_shared_runs(table, positions, page_size, self.MIN_KEYS)
        place = {row: at for at, row in enumerate(self.order)}
        group = n_q // n_kv
        spared = sum((len(run.rows) - 1) * (run.key_end - run.key_begin) for run in self.runs) * 2 * n_kv * head_dim * dtype.itemsize
        whole = (dtype == torch.bfloat16 and max(positions, default=0) < self.WHOLE_KEYS
                 and self.n_rows * n_kv * -(-group // self.FEW_COLUMNS) >= self.WHOLE_ROWS)
        self.pays = bool(self.runs) and spared >= self.PAYS_FROM and not whole
        # A run's columns in tiles of many, where there is work for them, and what is left, if that is little, in tiles of few.
        wide = dtype == torch.bfloat16 and head_dim in self.WIDE_HEADS
        size, little = (self.WIDE_COLUMNS, self.WIDE_LITTLE) if wide else (self.MANY_COLUMNS, self.MANY_LITTLE)
        scores = sum(len(run.rows) * (run.key_end - run.key_begin) for run in self.runs) * n_q
        if scores <= (self.WIDE_WORK if wide else self.MANY_WORK):
            little, target = self.n_rows * group, self.FEW_TARGET
        else:
            target = self.TARGET
        tiles = []                                        # per run: (first column, whether it is one of many)
        for run in self.runs:
            columns, at, found = len(run.rows) * group, 0, []
            while at < columns:
                many = columns - at > little
                found.append((at, many))
                at += size if many else self.FEW_COLUMNS
            tiles.append(found)
        # Parts of so many keys that all runs together make about the workgroups aimed at (no more: they would wait for a second round).
        work = sum(len(t) * (run.key_end - run.key_begin) for t, run in zip(tiles, self.runs)) * n_kv
        groups, parts_of = {False: [], True: []}, np.zeros(self.n_rows, dtype=np.int32)      # items that read the same keys and values
        for found, run in zip(tiles, self.runs):
            length = run.key_end - run.key_begin
            shortest, of_length = (self.MIN_WIDE_PART, length // 16) if wide and found[0][1] else (self.MIN_PART, length // WAVE)
            part = max(shortest, -(-work // target), min(of_length, self.LONG_PART))
            keys = -(-length // (32 * max(1, length // part))) * 32
            first = int(parts_of[run.rows[0]])
            for split, begin in enumerate(range(run.key_begin, run.key_end, keys)):
                end = min(run.key_end, begin + keys)
                for head in range(n_kv):
                    for kind in (False, True):
                        group_items = [(place[run.rows[0]], len(run.rows) * group, column, begin, end, first + split, run.rows[0], head)
                                       for column, many in found if many is kind]
                        if group_items:
                            groups[kind].append((end - begin, group_items))
            parts_of[run.rows] = first + -(-length // keys)
        items = {kind: self._in_order(some, fill) for kind, some in groups.items()}
        self.n_few, self.n_many = len(items[False]), len(items[True])
        self.shared_parts = int(parts_of.max(initial=0))
        self.own_begin = own_begin                        # int32 [B] on the host
        self.keys_end = max((run.key_end for run in self.runs), default=0)
        # A request's own keys in parts, the last of which has all that come behind it.
        ends = np.full(self.n_rows, table.shape[1] * self.page_size) if growth is None else np.asarray(positions, dtype=np.int64) + 1 + growth
        room = np.maximum(-(-ends // self.OWN_STEP) * self.OWN_STEP - own_begin, 1)
        longest, all_room = int(room.max(initial=1)), max(1, int(room.sum())) * n_kv * -(-group // self.FEW_COLUMNS)
        own_keys = max(self.MIN_PART, -(-longest // max(1, min(WAVE, self.OWN_TARGET * longest // all_room))))
        own_keys = -(-own_keys // 32) * 32
        own_parts = -(-room // own_keys)
        rows = np.arange(self.n_rows, dtype=np.int32)
        own_of_row = np.stack([rows, own_begin, parts_of, own_parts], axis=1).astype(np.int32)
        # (First parts of all requests first: the last ones are empty for the short ones.)
        own = [own_of_row[self.order]]
        for part in range(1, int(own_parts.max(initial=1))):
            with_it = own[0][own[0][:, 3] > part]
            own.append(with_it + np.array([0, part * own_keys, part, -part], dtype=np.int32))
        own = np.concatenate(own)
        self.n_own = self._filled(len(own), self.FILL_OWN if fill else 0)
        own = np.concatenate([own, np.full((self.n_own - len(own), 4), -1, dtype=np.int32)])
        self.slots = self._filled(int((parts_of + own_parts).max(initial=1)), self.FILL_SLOTS if fill else 0)
        packed = np.concatenate([np.asarray(items[False] + items[True], dtype=np.int32).reshape(-1), np.asarray(self.order, dtype=np.int32),
                                 own.reshape(-1), own_of_row.reshape(-1), np.array([own_keys], dtype=np.int32)]).astype(np.int32)
        self._on_device(torch.from_numpy(packed).to(device))

    # What a plan's counts are filled up to where it is to share captured graphs with others: the first of these doubled as often as it takes.  (Eight
    # answers that end one by one, behind 300 prompts of 64 to 8,000 tokens, 14 query heads: 189 graphs of steps, 524 with multiples of 32, 133
    # without plans.  What is filled in ends at once: 4 requests behind 512 keys 7.3 us instead of 6.9, 40 behind 4,096 20.2 instead of 19.7.)
    FILL_ITEMS, FILL_OWN, FILL_SLOTS = 256, 64, 16

    @staticmethod
    def _filled(count: int, least: int) -> int:
        if not least or not count:
            return count
        while least < count:
            least *= 2
        return least

    CHIPLETS = 8                  # of the device: each gets every eighth workgroup, and has a cache of its own

    @classmethod
    def _in_order(cls, groups, fill: bool) -> list[tuple]:
        """The items in the order of their workgroups: those of a group, which read the same keys and values, on one chiplet (two, where an
        even share of the work ends inside a group), the long ones first.  Places that a chiplet has left, and those up to a multiple of
        what `fill` asks for, hold items without columns."""
        queues = [[] for _ in range(cls.CHIPLETS)]
        # (A part's last piece may be a little shorter: shares are counted in eighths of the longest, so that equal parts stay equal.)
        step = max([1] + [-(-keys // 8) for keys, _ in groups])
        cost = lambda keys: -(-keys // step)
        total, before = sum(cost(keys) * len(group) for keys, group in groups), 0
        for keys, group in sorted(groups, key=lambda g: -g[0]):
            for item in group:
                queues[min(cls.CHIPLETS - 1, before * cls.CHIPLETS // total)].append(item)
                before += cost(keys)
        nothing = (0,) * 8
        longest = max(len(q) for q in queues)
        order = [queue[i] if i < len(queue) else nothing for i in range(longest) for queue in queues]
        while order and order[-1] is nothing:
            order.pop()
        return order + [nothing] * (cls._filled(len(order), cls.FILL_ITEMS if fill else 0) - len(order))

    def _on_device(self, packed: torch.Tensor) -> None:
        self.packed = packed
        sizes = [8 * (self.n_few + self.n_many), self.n_rows, 4 * self.n_own, 4 * self.n_rows, 1]
        self.items, self.order_dev, self.own_items, self.own_of_row_dev, self.own_keys_dev = torch.split(packed, sizes)
        self.own_dev = self.own_items[:4 * self.n_rows]                     # the requests' first parts
        self.places = tuple(4 * sum(sizes[:i]) for i in range(5))           # in bytes from the start of `packed`

    @property
    def signature(self) -> tuple:
        """What a launch depends on beside the tables: plans of one signature may take each other's place in a captured graph."""
        return (self.n_rows, self.n_few, self.n_many, self.n_own, self.slots, self.n_q, self.n_kv, self.head_dim, self.page_size, self.dtype)

    def standing_copy(self) -> "SharedPrefixes":
        """The same plan in memory of its own, which `take` fills with others of its signature (for a captured graph)."""
        copy = SharedPrefixes.__new__(SharedPrefixes)
        copy.__dict__.update(self.__dict__)
        copy._on_device(self.packed.clone())
        return copy

    def take(self, other: "SharedPrefixes") -> None:
        if other.signature != self.signature:
            raise ValueError("a plan of another make")
        self.order, self.runs, self.own_begin, self.keys_end = other.order, other.runs, other.own_begin, other.keys_end
        self.packed.copy_(other.packed, non_blocking=True)
