"""The page table of a batch in plain Python, from the words of include/mxfp4_hip.h (mxfp4_kv4_tables): which pages a
sequence has, a list of the free ones, and the tokens' places -- test infrastructure only."""
import numpy as np


class Tables:
    def __init__(self, B, max_pages, n_pages, page, window=None, sinks=0):
        self.page, self.window, self.sink_pages = page, window, -(-sinks // page)
        self.pages = np.full((B, max_pages), -1, np.int64)
        self.span = np.zeros((B, 2), np.int64)
        self.free = list(range(n_pages - 1, -1, -1))
        self.lacked = 0

    def has(self, lo, hi):
        return [i for i in range(hi) if i < self.sink_pages or i >= lo]

    def update(self, lens, news=None, T=0):
        B, max_pages = self.pages.shape
        room = max_pages * self.page
        wants, spans, olds, firsts = [], [], [], []
        self.lacked = 0
        for b in range(B):
            n = min(max(int(lens[b]), 0), room)
            hi, lo, gone_to = -(-n // self.page), 0, int(self.span[b, 0])
            olds.append(self.has(*self.span[b]))
            # all its positions are new, and pages are gone: it begins in the place of another
            anew = news is not None and 0 < n and int(lens[b]) <= int(news[b]) and gone_to > self.sink_pages
            first_taken = [i for i in range(self.sink_pages, min(gone_to, hi))][::-1] if anew else []
            if anew:
                gone_to = 0
            if self.window is not None:
                first = n - max(int(news[b]) if news is not None else 0, 0)        # the first position whose window counts
                needs = max(0, first - self.window + 1) // self.page
                lo = min(max(gone_to, needs), hi)
                self.lacked += len(set(self.has(needs, hi)) - set(self.has(lo, hi)))
            # pages past its row of the table
            n = max(int(lens[b]), 0)
            needs = 0
            if self.window is not None:
                needs = max(0, n - max(int(news[b]) if news is not None else 0, 0) - self.window + 1) // self.page
            past = range(max_pages, -(-n // self.page))
            if past:
                seen = range(max(needs, past.start), past.stop), range(past.start, min(self.sink_pages, needs, past.stop))
                self.lacked += sum(map(len, seen))
            spans.append((lo, hi))
            wants.append(self.has(lo, hi))
            firsts.append(first_taken)
        back = []
        for b in range(B):
            for i in olds[b]:
                if i not in wants[b]:
                    back.append(int(self.pages[b, i]))
                    self.pages[b, i] = -1
        self.free += back[::-1]                      # the r-th to place count + R - 1 - r
        for b in range(B):
            end = None
            for i in firsts[b] + [i for i in wants[b] if i not in firsts[b]]:
                if i in olds[b]:
                    continue
                if self.free:
                    self.pages[b, i] = self.free.pop()
                else:
                    self.lacked += 1
                    end = i if end is None else end
            lo, hi = spans[b]
            if end in firsts[b]:
                self.span[b] = end + 1, min(self.span[b, 1], hi)
            else:
                self.span[b] = (lo, hi) if end is None else (min(lo, end), end)
        if news is None:
            return None
        slots, seq, pos = [], [], []
        starts = [0]
        for b in range(B):
            for j in range(max(int(news[b]), 0)):
                p = int(lens[b]) - int(news[b]) + j
                pid = self.pages[b, p // self.page] if 0 <= p < room else -1
                slots.append(pid * self.page + p % self.page if pid >= 0 else -1)
                seq.append(b)
                pos.append(p)
            starts.append(len(seq))
        fill = [-1] * T
        return tuple(np.array((x + fill)[:T], np.int64) for x in (slots, seq, pos)) + (np.array(starts),)
