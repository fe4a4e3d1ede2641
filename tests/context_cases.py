"""Calls of the operators for long contexts with the kernel that takes them. test_context_edges_cpu.py asks the choice itself
whether that is so, so that a change of its estimates cannot take a kernel out of the GPU tests unseen."""
from collections import namedtuple

# kernel: "few" or "many"; cluster: blocks of a many-row cluster.
Window = namedtuple("Window", "sequences rows heads kv_heads tokens window sinks kernel cluster", defaults=(None,))
Prefix = namedtuple("Prefix", "sequences rows heads kv_heads prefix kernel cluster", defaults=(None,))

ALL = 1 << 20  # a window that holds everything

# What both kernels have to get right: scores far apart, NaN and infinities in sight, outputs over queries, strides.
FEW = Window(2, 9, 12, 4, 700, 500, 3, "few")
MANY = Window(2, 300, 12, 4, 3000, 2000, 3, "many", 4)
MANY_ALONE = Window(4, 300, 16, 4, 2000, 1500, 70, "many", 1)         # no cluster, odd last query tile
MANY_ONE_TILE = Window(24, 32, 32, 8, 2048, ALL, 0, "many", 1)        # both halves of a block share its only query tile
MANY_OF_256 = Window(1, 40, 256, 1, 3000, 2500, 4, "many", 2)         # 256 query heads over one
MANY_OF_64 = Window(2, 20, 64, 1, 5000, 4000, 4, "many", 8)
MANY_LOADED = Window(2, 300, 28, 4, 3000, ALL, 0, "many", 2)          # groups of seven: no box copies their queries
MANY_SHORT = Window(1, 129, 16, 4, 4000, 3000, 0, "many", 8)          # five query tiles, the last of one row

HARD = dict(few=FEW, many=MANY, many_alone=MANY_ALONE, many_one_tile=MANY_ONE_TILE, many_of_256=MANY_OF_256, many_of_64=MANY_OF_64,
            many_loaded=MANY_LOADED, many_short=MANY_SHORT)

# Waits that run out: few rows in clusters, without, in two units a head, eight warps, two row tiles; many rows as above.
GIVE_UP = dict(few_clusters=Window(2, 1, 8, 8, 3000, ALL, 0, "few"), few_alone=Window(40, 1, 32, 8, 90, ALL, 0, "few"),
               few_two_units=Window(2, 5, 28, 4, 700, ALL, 0, "few"), few_long=Window(2, 2, 8, 2, 9000, ALL, 0, "few"),
               few_64=Window(2, 16, 32, 8, 4000, ALL, 0, "few"), many_loaded=MANY_LOADED, many=Window(3, 700, 32, 8, 2000, ALL, 0, "many", 1),
               many_one_tile=MANY_ONE_TILE, many_short=Window(1, 129, 16, 4, 4000, ALL, 0, "many", 8), many_of_256=Window(1, 40, 256, 1, 3000, ALL, 0, "many", 2))

# In a graph whose lengths change.
GRAPH = dict(few=Window(2, 3, 16, 4, 300, 90, 4, "few"), many=Window(2, 260, 16, 4, 3000, 2500, 4, "many", 2))

PREFIX_GIVE_UP = dict(few=Prefix(2, 1, 8, 2, 900, "few"), many=Prefix(64, 1, 32, 8, 8192, "many", 4), many_odd=Prefix(3, 40, 28, 4, 9001, "many", 1))
PREFIX_HARD = dict(few=Prefix(3, 2, 8, 2, 900, "few"), many=Prefix(64, 1, 32, 8, 8192, "many", 4), many_rows=Prefix(3, 300, 12, 4, 4000, "many", 1))
