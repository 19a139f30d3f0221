"""A plain form of the page pool: sequences one after the other, in Python's numbers."""


def pages_of(n, page):
    return -(-n // page)


class PlainPool:
    def __init__(self, uses, page, table, lengths):
        self.uses, self.page = list(uses), page
        self.table, self.lengths = [list(r) for r in table], list(lengths)
        self.starts = [0] * (len(lengths) + 1)

    def extend(self, new, rows):
        page, width = self.page, len(self.table[0]) if self.table else 0
        free = [p for p, n in enumerate(self.uses) if n <= 0]
        asked_rows = asked_pages = at = 0
        slots, positions, self.starts = [], [], [0]
        for i, n in enumerate(new):
            n, old = max(n, 0), max(self.lengths[i], 0)
            have = pages_of(old, page)
            need = pages_of(old + n, page) - have
            room = old + n <= width * page
            if room:
                asked_rows, asked_pages = asked_rows + n, asked_pages + need
            if room and asked_rows <= rows and (need == 0 or asked_pages <= len(free)):
                for w in range(have, have + need):
                    self.table[i][w] = free[at]
                    self.uses[free[at]] = 1
                    at += 1
                if n > 0:
                    self.lengths[i] = old + n
                for p in range(old, old + n):
                    at_page = self.table[i][p // page]
                    there = 0 <= at_page < len(self.uses)
                    slots.append(at_page * page + p % page if there else -1)
                    positions.append(p)
            self.starts.append(len(positions))
        rest = [-1] * (rows - len(positions))
        return slots + rest, positions + rest

    def release(self, lengths=None, window=None, sinks=0):
        page = self.page
        for i, row in enumerate(self.table):
            old = max(self.lengths[i], 0)
            to = old if lengths is None else min(max(lengths[i], 0), old)
            for w in range(min(pages_of(old, page), len(row))):
                past = w >= pages_of(to, page)
                left = window is not None and (w + 1) * page - 1 <= to - window and w * page >= sinks
                if (past or left) and 0 <= row[w] < len(self.uses):
                    self.uses[row[w]] -= 1
                    row[w] = -1
            if lengths is not None:
                self.lengths[i] = to
