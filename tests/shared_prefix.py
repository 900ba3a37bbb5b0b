"""Problems for the operators of a batch that shares a long prefix, and their definitions in 64-bit torch."""
import math

import torch

PAGE = 64
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}          # half a step, relative to the value


def axis_of(sections, interleaved):
    n = len(sections)
    if not interleaved:
        return [a for a, count in enumerate(sections) for _ in range(count)]
    return [i % n if i < n * sections[i % n] else 0 for i in range(sum(sections))]


def turned(x, positions, denom, sections, interleaved=False, neighbours=False):
    """x [rows, heads, hd] double, with its pairs turned, and the bound on a 32-bit computation's error before the last rounding.

    The bound, per number: (|a| + |b|) times the error of a sine or cosine and of the two products and their sum.  The angle is a
    fraction of a half turn rounded to 32-bit (pi 2^-24), plus what a step in double precision leaves at position p (p 2^-52); sine and
    cosine are off by at most two units (2 * 2^-23 = 4 * 2^-24), the products and the sum by 2^-24 each."""
    half = sum(sections)
    out, err = x.clone(), torch.zeros_like(x)
    for i, a in enumerate(axis_of(sections, interleaved)):
        pos = positions[:, a].double()
        angle = (pos / float(denom[i]))[:, None]
        f, s = (2 * i, 2 * i + 1) if neighbours else (i, i + half)
        out[:, :, f] = x[:, :, f] * angle.cos() - x[:, :, s] * angle.sin()
        out[:, :, s] = x[:, :, s] * angle.cos() + x[:, :, f] * angle.sin()
        slack = (x[:, :, f].abs() + x[:, :, s].abs()) * ((math.pi + 4 + 2) * 2.0 ** -24 + pos.abs() * 2.0 ** -52)[:, None]
        err[:, :, f] = slack
        err[:, :, s] = slack
    return out, err


class Geometry:
    def __init__(self, starts, q_lens, max_kv_len, device):
        self.n_seqs, self.max_q_len, self.max_kv_len = len(q_lens), max(max(q_lens), 1), max_kv_len
        self.decode = self.max_q_len == 1
        self.seq_start = torch.tensor(starts, dtype=torch.int32, device=device)
        self.seq_qlen = torch.tensor(q_lens, dtype=torch.int32, device=device)


class Batch:
    """Sequences of own_lens keys behind a prefix, the last q_lens of them this step's rows.  Pages are shuffled over the pool; what
    no sequence holds, and the rows behind a sequence's end, are NaN."""

    def __init__(self, dtype, q_lens, own_lens, prefix, heads, kv_heads, hd, window=0, seed=0, device="cuda:0", spread=1.5, beside=0,
                 wider=0, pool_extra=3, page=PAGE):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.heads, self.kv_heads, self.hd, self.window, self.prefix, self.device = dtype, heads, kv_heads, hd, window, prefix, device
        self.q_lens, self.own_lens = q_lens, own_lens
        self.page = size = page
        rows = sum(q_lens)
        counts = [-(-prefix // size)] + [-(-n // size) for n in own_lens]
        pages = sum(counts) + pool_extra
        perm = torch.randperm(pages, generator=g).tolist()
        self.k_pool = torch.full((pages, size, kv_heads, hd), float("nan"), dtype=dtype, device=device)
        self.v_pool = self.k_pool.clone()
        width = max(counts[1:]) + wider
        at, tables = 0, []
        for c in counts:
            tables.append(perm[at:at + c])
            at += c
        for table, n in zip(tables, [prefix] + own_lens):
            for lp, page in enumerate(table):
                here = min(size, n - lp * size)
                self.k_pool[page, :here] = torch.randn((here, kv_heads, hd), generator=g).to(dtype).to(device)
                self.v_pool[page, :here] = torch.randn((here, kv_heads, hd), generator=g).to(dtype).to(device)
        self.prefix_table = torch.tensor(tables[0], dtype=torch.int32, device=device)
        self.block_table = torch.tensor([t + [-1] * (width - len(t)) for t in tables[1:]], dtype=torch.int32, device=device).view(len(q_lens), width)
        # the queries' rows may be part of wider ones
        self.wide = (torch.randn((rows, beside + heads * hd + beside), generator=g) * spread).to(dtype).to(device)
        self.q = self.wide[:, beside:beside + heads * hd] if beside else self.wide
        self.row_seq = torch.tensor([s for s, q in enumerate(q_lens) for _ in range(q)], dtype=torch.int32, device=device)
        self.row_pos = torch.tensor([prefix + n - q + t for q, n in zip(q_lens, own_lens) for t in range(q)], dtype=torch.int32, device=device)
        starts = [sum(q_lens[:s]) for s in range(len(q_lens))]
        self.geometry = Geometry(starts, q_lens, prefix + max(own_lens), device)
        self.scale = hd ** -0.5
        self.out = torch.full((rows, heads * hd), 7.25, dtype=dtype, device=device)

    def run(self, ops, out=None):
        out = self.out if out is None else out
        ops.attention_shared(self.q, self.wide.stride(0), out, self.k_pool, self.v_pool, self.prefix_table, self.prefix, self.block_table,
                             self.page, self.row_seq, self.row_pos, self.heads, self.kv_heads, self.hd, self.window, self.scale, self.geometry)
        return out

    def reference(self):
        """(result [rows, heads * hd], bound on the error of a correct kernel), both double.

        The bound, with A = sum_j w_j |v_j| / sum_j w_j (w: weights): scores are sums of hd products in 32-bit, off by at most
        delta = (hd + 4) 2^-24 scale sum |q k| each, which changes a weight by the factor 1 + delta and so a result by 2 delta A; an
        exponential adds 2^-21; sums over n keys and parts in 32-bit n 2^-24; weights rounded to the result's type before they meet
        the values half a step of it (bf16; none in float32); the result is rounded once."""
        rows, group, device = self.q.shape[0], self.heads // self.kv_heads, self.device
        out = torch.zeros((rows, self.heads, self.hd), dtype=torch.float64, device=device)
        tol = torch.zeros_like(out)
        q_all = self.q.double().view(rows, self.heads, self.hd)
        kf, vf = self.k_pool.double().flatten(0, 1), self.v_pool.double().flatten(0, 1)
        half = HALF[self.dtype]
        for r in range(rows):
            seq, pos = int(self.row_seq[r]), int(self.row_pos[r])
            if seq < 0:
                continue
            room = self.prefix + self.block_table.shape[1] * self.page
            lo = max(0, pos - self.window + 1) if self.window > 0 else 0
            j = torch.arange(lo, min(pos, room - 1) + 1, device=device)
            if j.numel() == 0:
                continue
            own = j - self.prefix
            table_p = self.prefix_table.long() if self.prefix_table.numel() else torch.zeros(1, dtype=torch.long, device=device)
            table_o = self.block_table[seq].long() if self.block_table.shape[1] else torch.zeros(1, dtype=torch.long, device=device)
            page = torch.where(own < 0, table_p[(j // self.page).clamp(max=table_p.numel() - 1)], table_o[(own // self.page).clamp(0, table_o.numel() - 1)])
            place = torch.where(own < 0, j, own) % self.page
            named = (page >= 0) & (page < self.k_pool.shape[0])
            flat = page.clamp(0, self.k_pool.shape[0] - 1) * self.page + place
            k = torch.where(named[:, None, None], kf[flat], 0.0)
            v = torch.where(named[:, None, None], vf[flat], 0.0)
            for h in range(self.kv_heads):
                q = q_all[r, h * group:(h + 1) * group]
                score = q @ k[:, h].T * self.scale
                w = torch.softmax(score, -1)
                delta = (self.hd + 4) * 2.0 ** -24 * self.scale * (q.abs() @ k[:, h].abs().T).amax(-1, keepdim=True)
                around = w @ v[:, h].abs()
                o = w @ v[:, h]
                out[r, h * group:(h + 1) * group] = o
                tol[r, h * group:(h + 1) * group] = half * o.abs() + around * (
                    2 * delta + 2.0 ** -21 + (j.numel() + 64) * 2.0 ** -24 + (half if self.dtype != torch.float32 else 0.0)) + 1e-30
        return out.flatten(1), tol.flatten(1)

    def check(self, out, what=""):
        ref, tol = self.reference()
        live = self.row_seq >= 0
        err = (out.double() - ref).abs()
        bad = ~(err <= tol) & live[:, None]
        assert not bool(bad.any()), "%s: %d numbers off, the worst by %.3g of the bound (row %d)" % (
            what, int(bad.sum()), float((err / tol)[bad].nan_to_num(1e9).max()), int(bad.nonzero()[0, 0]))
        assert bool((out[~live] == 7.25).all()), "%s: a row without a sequence was written" % what
