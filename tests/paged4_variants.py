"""Calls of attention over pages of 4 bits for each form of its kernel of few rows: tiles of 4
rows (four key blocks a step), and of 8 by eight or four wavefronts, whole or split."""
from dataclasses import dataclass

PAGE = 64


@dataclass(frozen=True)
class Call:
    form: tuple  # rows of a tile, eight wavefronts?, split?
    heads: int
    kv_heads: int
    d: int
    lengths: tuple  # of the sequences, the new rows included
    new: tuple
    window: int | None = None
    sinks: int = 0

    def __str__(self):
        return (f"{self.heads}on{self.kv_heads}x{self.d}-{len(self.new)}x{max(self.new)}of{sum(self.new)}-"
                f"after{max(self.lengths)}-{self.window}+{self.sinks}")

    @property
    def width(self):
        return -(-max(self.lengths) // PAGE)


FOUR, WIDE, WIDE_SPLIT, EIGHT, EIGHT_SPLIT = ((4, True, False), (8, True, False), (8, True, True),
                                              (8, False, False), (8, False, True))
WINDOWS = ((None, 0), (1000, 0), (2048, 4), (1000, 70), (2048, 70))

CALLS = []
for d in (64, 96, 128):
    # rows of one token on 1, 3 and 4 heads; of several, in one tile and in two; idle sequences
    for heads, new in ((8, (1,)), (6, (1,)), (2, (1,)), (8, (1, 1, 1)), (6, (1, 0, 1)), (2, (4,)), (2, (3, 1, 0)),
                       (4, (2,)), (4, (1, 2, 2)), (4, (4, 1, 0, 1)), (2, (2, 1, 9, 4, 1, 1, 5, 1))):
        lengths = (2100, 801, 1500, 1023, 1, 64, 2081, 900)[:len(new)]
        for window, sinks in WINDOWS:
            CALLS.append(Call(FOUR, heads, 2, d, lengths, new, window, sinks))
    # the last blocks of a wavefront's step missing, by one to three; steps of one block
    for length in (769, 800, 1024, 1025, 1056, 1057, 1088, 1120, 2048, 2049):
        CALLS.append(Call(FOUR, 8, 2, d, (length,), (1,)))
    CALLS.append(Call(FOUR, 8, 2, d, (2000,) * 95 + (37,), (1,) * 96, 2000, 4))
    for window, sinks in ((None, 0), (1000, 0), (1000, 70)):
        CALLS.append(Call(WIDE, 16, 2, d, (1030,), (1,), window, sinks))
        CALLS.append(Call(WIDE, 16, 2, d, (1030, 3, 900, 777), (1, 1, 1, 1), window, sinks))
        CALLS.append(Call(WIDE, 8, 2, d, (1100, 1024), (2, 2), window, sinks))
        CALLS.append(Call(WIDE, 6, 2, d, (1100, 900, 1000), (2, 3, 0), window, sinks))
    for window, sinks in ((None, 0), (5000, 0), (4900, 300)):
        CALLS.append(Call(WIDE_SPLIT, 64, 8, d, (6000, 1200, 5500, 20), (1, 1, 1, 1), window, sinks))
    for window, sinks in ((None, 0), (8300, 0), (8250, 300)):
        CALLS.append(Call(WIDE_SPLIT, 8, 8, d, (9000, 1200), (6, 8), window, sinks))
    for window, sinks in ((None, 0), (300, 0), (300, 100)):
        CALLS.append(Call(EIGHT, 8, 2, d, (700, 500, 33), (1, 1, 1), window, sinks))
        CALLS.append(Call(EIGHT, 5, 1, d, (600, 90), (1, 2), window, sinks))
    for window, sinks in ((None, 0), (2500, 0), (2500, 70)):
        CALLS.append(Call(EIGHT_SPLIT, 16, 2, d, (3000, 900), (1, 1), window, sinks))
        CALLS.append(Call(EIGHT_SPLIT, 6, 2, d, (3000, 900, 2800), (2, 3, 1), window, sinks))

# For tests of their own: (heads, new rows, length, form) of one sequence on 2 kv heads, with
# these windows.
UNSEEN = ((8, 1, 1500, FOUR), (6, 1, 1217, FOUR), (4, 2, 1500, FOUR), (2, 4, 1290, FOUR), (16, 1, 1050, WIDE),
          (8, 2, 1050, WIDE))
UNSEEN_WINDOWS = ((None, 0), (1000, 0), (1000, 70), (998, 78))
STALE = 40  # positions behind the length
MISSING = ((8, 1, 1101, FOUR), (6, 1, 1101, FOUR), (2, 3, 1103, FOUR), (16, 1, 1101, WIDE), (6, 2, 1102, WIDE))
MISSING_WINDOWS = ((None, 0), (1000, 0), (1000, 70))
