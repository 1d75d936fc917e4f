"""Shapes of the paged attention, one or more for every kernel that its plans choose:
the CPU test of the plans checks that each still gets the kernel it stands for, the
GPU tests run it.  Pages have 16 rows."""

PAGE = 16

# Prompts: head size, bytes a value, runs of new tokens (all of their own keys), shared
# keys, kv heads, query heads of each, unused pages a table has beyond the longest run;
# 64 rt rows a block (0: 16), streams of keys a block, whether the keys are in parts.
PROMPTS = [
    (64, 2, [17], 390, 1, 1, 1, 0, 1, False),
    (64, 2, [17], 1000, 1, 16, 200, 0, 1, True),
    (64, 2, [49, 31], 390, 8, 16, 1, 1, 1, False),
    (64, 2, [17], 1000, 1, 1, 200, 1, 1, True),
    (64, 2, [76, 67, 58], 77, 4, 16, 200, 1, 2, False),
    (64, 2, [99, 90, 81], 390, 8, 16, 1, 2, 1, False),
    (64, 2, [67], 1000, 4, 8, 200, 2, 1, True),
    (64, 2, [49, 40, 31], 77, 8, 16, 200, 2, 2, False),
    (64, 2, [40], 1000, 8, 16, 200, 2, 2, True),
    (64, 4, [17], 390, 1, 1, 1, 0, 1, False),
    (64, 4, [17], 1000, 1, 1, 1, 0, 1, True),
    (64, 4, [49, 31], 200, 8, 16, 1, 1, 1, False),
    (64, 4, [17], 1000, 8, 7, 200, 1, 1, True),
    (64, 4, [76, 58], 77, 8, 16, 1, 1, 2, False),
    (64, 4, [139, 130, 121], 390, 8, 16, 200, 2, 1, False),
    (64, 4, [49, 31], 1000, 8, 8, 200, 2, 1, True),
    (64, 4, [99, 90, 81], 200, 8, 16, 1, 2, 2, False),
    (128, 2, [17], 390, 1, 1, 1, 0, 1, False),
    (128, 2, [17], 1000, 1, 3, 200, 0, 1, True),
    (128, 2, [67], 390, 8, 16, 1, 1, 1, False),
    (128, 2, [17], 1000, 1, 1, 1, 1, 1, True),
    (128, 2, [49, 31], 200, 8, 16, 200, 1, 2, False),
    (128, 2, [17], 1000, 8, 16, 200, 1, 2, True),
    (128, 2, [99, 90, 81], 390, 8, 16, 1, 2, 1, False),
    (128, 2, [26, 17, 8], 1000, 8, 4, 200, 2, 1, True),
    (128, 2, [49, 40, 31], 390, 8, 16, 200, 2, 2, False),
    (128, 2, [67], 1000, 8, 8, 200, 2, 2, True),
    (128, 4, [17], 200, 1, 1, 1, 0, 1, False),
    (128, 4, [17], 1000, 1, 1, 1, 0, 1, True),
    (128, 4, [49, 31], 77, 8, 16, 1, 1, 1, False),
    (128, 4, [17], 1000, 8, 7, 200, 1, 1, True),
    (128, 4, [76, 58], 200, 8, 16, 1, 1, 2, False),
    (128, 4, [40], 1000, 2, 16, 200, 1, 2, True),
    (256, 2, [17], 200, 1, 1, 1, 0, 1, False),
    (256, 2, [17], 1000, 1, 3, 200, 0, 1, True),
    (256, 2, [67], 77, 8, 16, 1, 1, 1, False),
    (256, 2, [17], 1000, 1, 1, 1, 1, 1, True),
    (256, 2, [90], 390, 8, 16, 200, 1, 2, False),
    (256, 2, [17], 1000, 4, 16, 200, 1, 2, True),
    (256, 4, [17], 77, 1, 1, 1, 0, 1, False),
    (256, 4, [17], 1000, 1, 7, 200, 0, 1, True),
    (256, 4, [26, 17, 8], 77, 8, 16, 1, 1, 1, False),
    (256, 4, [17], 1000, 1, 1, 1, 1, 1, True),
]


def prompt_plan_args(hd, size, runs, prefix, n_kv, rep, room):
    capacity = (-(-max(runs) // PAGE) + room) * PAGE
    return hd * size, hd, n_kv, rep, prefix, capacity, len(runs), sum(runs)


# One token a sequence: bytes a value, own lengths, shared keys, query heads of each of
# two kv heads, unused pages; the same rt of the shared keys' rows by head size (64,
# 128, 256), whether the shared keys and the own ones are in parts.
_UNEVEN = [0, 1, 777, 16, 300] + [3 * i % 41 for i in range(35)]
DECODES = [
    (2, _UNEVEN[:5], 1100, 3, 1, (0, 0, 0), True, True),
    (2, _UNEVEN[:15], 1100, 3, 1, (1, 1, 1), True, True),
    (2, _UNEVEN, 1100, 3, 1, (2, 2, 1), True, True),
    (4, _UNEVEN[:5], 1100, 3, 1, (0, 0, 0), True, True),
    (4, _UNEVEN[:15], 1100, 3, 1, (1, 1, 1), True, True),
    (4, _UNEVEN, 1100, 3, 1, (2, 1, 1), True, True),
    # tables a hundred times as wide as the lengths
    (2, [5, 0, 33], 40, 4, 500, (0, 0, 0), None, True),
    (4, [5, 0, 33], 40, 4, 500, (0, 0, 0), None, True),
    (2, [900, 40] + [20] * 30, 40, 4, 2000, (2, 2, 1), None, True),
    # no own keys at all
    (2, [0] * 40, 1100, 3, 0, (2, 2, 1), True, False),
    (4, [0] * 40, 1100, 3, 0, (2, 1, 1), True, False),
    (2, [0] * 3, 1100, 2, 0, (0, 0, 0), True, False),
]


def decode_plan_args(hd, size, lens, prefix, rep, room):
    capacity = (-(-max(lens) // PAGE) + room) * PAGE
    return hd * size, hd, 2, rep, prefix, capacity, len(lens)


# Thousands of rows of more than 16 parts: (bytes a value, own lengths, shared keys, query
# heads of each of two kv heads, unused pages).
MERGES = [(2, [777, 0, 5, 33] * 16, 1100, 32, 2000), (4, [777, 0, 5, 33] * 16, 1100, 32, 2000)]

# The same for few keys: one block a sequence and kv head takes prefix and own ones
# together (by head size), or parts do because the batch is large.
JOINTS = [
    (2, [3, 0, 18], 12, 3, 1, (1, 1, 1)),
    (4, [3, 0, 18], 12, 3, 1, (1, 1, 1)),
    (2, [200, 0, 31], 12, 20, 1, (1, 1, 1)),
    (2, [90, 0, 31], 0, 3, 1, (1, 1, 1)),
    (4, [60, 0, 31], 30, 3, 1, (1, 1, 1)),
    (2, [3, 16, 0, 9] * 256, 210, 1, 0, (1, 0, 0)),
    (4, [3, 16, 0, 9] * 128, 210, 1, 0, (1, 0, 0)),
    (4, [3, 16, 0, 9] * 128, 470, 1, 0, (0, 0, 0)),
    (2, [3, 16, 0, 9] * 256, 930, 1, 0, (0, 0, 0)),
]
