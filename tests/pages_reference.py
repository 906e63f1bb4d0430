"""The pages of a cache as the header defines them, row by row and page by page."""


def entries(tokens, page):
    return -(-tokens // page)


class Pages:
    def __init__(self, pages, rows, table_pages, page):
        self.pages, self.rows, self.table_pages, self.page = pages, rows, table_pages, page
        self.refs, self.lens = [0] * pages, [0] * rows
        self.table = [[-1] * table_pages for _ in range(rows)]

    def counted(self, p):
        return 0 <= p < self.pages

    def update(self, parents=None, add=None):
        """(rows that did not grow, copies [(from, to)])"""
        table, lens = [list(r) for r in self.table], list(self.lens)
        begin = []
        for b in range(self.rows):
            p = b if parents is None else parents[b]
            p = p if 0 <= p < self.rows else None
            had = 0 if p is None else lens[p]
            want = max(0, had + (add[b] if add is not None else 0))
            kept = entries(min(had, want), self.page)
            begin.append((had, want, [] if p is None else table[p][:kept]))
        for b in range(self.rows):   # what the rows had, and what they begin with
            for x in table[b][:entries(lens[b], self.page)]:
                if self.counted(x):
                    self.refs[x] -= 1
            for x in begin[b][2]:
                if self.counted(x):
                    self.refs[x] += 1
        shared = {x for x in range(self.pages) if self.refs[x] > 1}
        free = [x for x in range(self.pages) if self.refs[x] == 0]
        short, copies, enough = [0] * self.rows, [], True
        for b, (had, want, row) in enumerate(begin):
            now, row = want, list(row)
            if want > had:
                torn = row[had // self.page] if had % self.page else -1
                torn = torn if self.counted(torn) and torn in shared else -1
                need = entries(want, self.page) - len(row) + (torn >= 0)
                if want > self.table_pages * self.page:
                    now, short[b] = had, 1
                elif not enough or need > len(free):
                    enough = False
                    now, short[b] = had, 1
                else:
                    taken, free = free[:need], free[need:]
                    if torn >= 0:
                        copies.append((torn, taken[0]))
                        self.refs[torn] -= 1
                        row[-1] = taken.pop(0)
                        self.refs[row[-1]] = 1
                    for x in taken:
                        self.refs[x] = 1
                        row.append(x)
            self.table[b], self.lens[b] = row + [-1] * (self.table_pages - len(row)), now
        return short, copies

    def compact(self):
        """(pages in use, moves [(from, to)], where every page is now)"""
        used = [x for x in range(self.pages) if self.refs[x]]
        n = len(used)
        moves = list(zip([x for x in used if x >= n], [x for x in range(n) if not self.refs[x]]))
        to = {a: b for a, b in moves}
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(x, x) for x in row] for row in self.table]
        moved = [-1] * self.pages
        for x in used:
            moved[x] = to.get(x, x)
        return n, moves, moved
