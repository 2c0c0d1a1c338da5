"""CPU replay of the attention kernels' line of tiles (go-infer_b200/csrc/paged.cuh, run_of_line and the walk over
a run's units) and of the merge's places on it (paged_attn.cu, attn_merge_kernel)."""


def seq_of(b, q_start, kv_len, n_tokens, prefix=0):
    """(start, fresh, len) of sequence b, or of the prefix as one sequence."""
    first, last = (0, len(q_start) - 1) if prefix else (b, b + 1)
    start = max(0, min(q_start[first], n_tokens))
    fresh = max(start, min(q_start[last], n_tokens)) - start
    return start, fresh, prefix or max(0, kv_len[b])


class Line:
    """A pass: its sequences' places, the places per CTA, and each CTA's units."""

    def __init__(self, q_start, kv_len, n_tokens, group, kv_heads, rows, tt, unit_cost, ctas, least, prefix=0):
        self.rows, self.tt, self.cost, self.group, self.kv_heads, self.prefix = rows, tt, unit_cost, group, kv_heads, prefix
        self.seqs = [seq_of(b, q_start, kv_len, n_tokens, prefix) for b in range(1 if prefix else len(kv_len))]
        self.spans, self.first, at = [], [], 0
        for _, fresh, n in self.seqs:
            rt, tl = -(-fresh * group // rows), max(1, -(-n // tt))
            self.spans.append((rt, tl, tl + unit_cost))
            self.first.append(at)
            at += rt * (tl + unit_cost) * kv_heads
        self.total, self.ctas = at, ctas
        self.chunk = max(-(-at // ctas), least)

    def seen(self, s, j):
        _, fresh, n = s
        return n if self.prefix else max(0, min(n, n - fresh + j + 1))

    def units(self, cta):
        """The units of a CTA's run: (sequence, kv head, first row, first tile, tiles of the run, tiles that a row sees)."""
        pos, end = cta * self.chunk, min(self.total, (cta + 1) * self.chunk)
        out = []
        while pos < end:
            b = max(i for i, f in enumerate(self.first) if f <= pos and self.spans[i][0])
            rt, tl, unit = self.spans[b]
            u, at0 = divmod(pos - self.first[b], unit)
            at1 = min(at0 + end - pos, unit)
            pos += at1 - at0
            tile0 = max(at0 - self.cost, 0)
            count = at1 - self.cost - tile0
            if count <= 0:
                break
            row0 = u % rt * self.rows
            n_rows = min(self.rows, self.seqs[b][1] * self.group - row0)
            last = self.seen(self.seqs[b], (row0 + n_rows - 1) // self.group)
            out.append((b, u // rt, row0, tile0, count, max(0, min(tile0 + count, -(-last // self.tt)) - tile0)))
        return out

    def parts(self, token, h, hg, b=0):
        """(row of the unit, CTAs of the unit that holds row (token, head), their slots), as the merge computes them."""
        start, _, _ = self.seqs[b]
        rt, tl, unit = self.spans[b]
        row = (token - start) * self.group + hg
        u1 = self.first[b] + (h * rt + row // self.rows + 1) * unit
        u0 = u1 - tl
        i0, i1 = u0 // self.chunk, (u1 - 1) // self.chunk
        return row % self.rows, [(i, 0 if i * self.chunk > u0 else 1) for i in range(i0, i1 + 1)]
