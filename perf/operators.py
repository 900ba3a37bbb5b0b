"""Operators of serving many continuations of one long document, image or video, alone: the rotation of heads by positions
with several axes, the same with keys and values appended to the paged cache, and attention of a batch that shares a long
prefix.

A case is one call; "op" names the operator:
  "rotate"   heads of every row are turned by the row's positions (two axes: patches of an image; three: time, height, width);
  "append"   queries are turned, keys are turned on their way into the cache's pages, values go there as they are;
  "shared"   a batch of sequences with one prefix: their rows against the prefix' pages and each sequence's own.
Head layouts are those of this repository's models (28 heads on 4 of 128, 40 on 8 of 128, 3 on 1 of 32) and generic ones; a
vision tower has as many key heads as query heads, 16 of 80.  `run` states each operator in elementary 32-bit torch (angles in
64-bit), or, with `own`, calls the library.  `exact` states them in 64-bit.
"""
import math

import torch

own = False

PAGE = 64
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}

# The widest pass of each operator, in the unit that its cost goes by; drawn cases stay within it.
ROTATE_ELEMENTS = 65536 * 32 * 80
APPEND_ELEMENTS = 32770 * 56 * 128
SHARED_FLOPS, SHARED_BYTES = 2.3e11, 9.8e7
SHARED_FLOPS_F32 = 1.2e9
SHARED_SCORES = 5.0e8           # and what the plain form keeps of scores, for the prefix and for the padded own keys


def listed():
    bf, f32 = "bfloat16", "float32"
    return [
        # q and k of one small image's 256 patches in a vision tower (the values lie beside them and stay)
        rotate_case("rotate_image_256", bf, 256, 32, 80, [20, 20], beside=16),
        # q and k of a long video clip's patches, 32-bit checks of such a tower's rotation, and the clip in bf16
        rotate_case("rotate_patches_2311_f32", f32, 2311, 32, 80, [20, 20], beside=16, neighbours=True),
        rotate_case("rotate_clip_65536", bf, 65536, 32, 80, [20, 20], beside=0),
        # one more token for each of eight sequences: latency
        append_case("append_decode_8", bf, [1] * 8, 28, 4, 128, [16, 24, 24], [5000, 40, 777, 63, 64, 1999, 3, 900]),
        # an image of 4,099 tokens and a question to it, in two sequences
        append_case("append_image_4099", bf, [4099, 37], 28, 4, 128, [16, 24, 24], [0, 4100]),
        # a video of 32,770 tokens, heads of 40 on 8, axes dealt out to the frequencies in turn
        append_case("append_video_32770", bf, [32770], 40, 8, 128, [24, 20, 20], [0], interleaved=True),
        # the 32-bit path: three prompts of unequal lengths
        append_case("append_prompts_f32", f32, [701, 1, 829], 14, 2, 64, [8, 12, 12], [0, 65, 10]),
        # a short shared instruction, four sequences: latency
        shared_case("shared_decode_4", bf, [1] * 4, 500, [1, 40, 17, 33], 14, 2, 64),
        # sixteen answers to one document
        shared_case("shared_decode_16", bf, [1] * 16, 4000, [17 * i % 301 + 1 for i in range(16)], 28, 4, 128),
        # sixty-four answers to a long one
        shared_case("shared_decode_64", bf, [1] * 64, 16001, [157 * i % 1000 + 1 for i in range(64)], 28, 4, 128),
        # sixteen questions of unequal lengths to the same document, taken in at once
        shared_case("shared_prompts_16", bf, [16 + 53 * i % 241 for i in range(16)], 8000, [16 + 53 * i % 241 for i in range(16)], 28, 4, 128),
        # the 32-bit path: eight answers
        shared_case("shared_decode_8_f32", f32, [1] * 8, 1500, [13 * i % 97 + 1 for i in range(8)], 14, 2, 64),
    ]


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def _lists(case):
    """The case with its lists as lists (a case itself holds plain values only)."""
    return {k: [int(n) for n in v.split(",")] if k in ("sections", "q_lens", "pos0", "own_lens") else v for k, v in case.items()}


def rotate_case(name, dtype, rows, heads, hd, sections, beside=0, interleaved=False, neighbours=False):
    """beside: further heads of the same rows that lie behind the rotated ones and are not touched."""
    return {"name": name, "op": "rotate", "dtype": dtype, "rows": rows, "heads": heads, "hd": hd, "sections": _text(sections),
            "beside": beside, "interleaved": interleaved, "neighbours": neighbours}


def append_case(name, dtype, q_lens, heads, kv_heads, hd, sections, pos0, interleaved=False, neighbours=False):
    """q_lens: new tokens of each sequence; pos0: what its cache holds before them."""
    return {"name": name, "op": "append", "dtype": dtype, "q_lens": _text(q_lens), "heads": heads, "kv_heads": kv_heads,
            "hd": hd, "sections": _text(sections), "pos0": _text(pos0), "interleaved": interleaved, "neighbours": neighbours}


def shared_case(name, dtype, q_lens, prefix, own_lens, heads, kv_heads, hd, window=0):
    """own_lens: keys of each sequence behind the prefix, the new tokens' included."""
    return {"name": name, "op": "shared", "dtype": dtype, "q_lens": _text(q_lens), "prefix": prefix, "own_lens": _text(own_lens),
            "heads": heads, "kv_heads": kv_heads, "hd": hd, "window": window}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _sections(rng, half, axes):
    """`half` pairs dealt out to the axes such that they may also be dealt in turn (no later axis has more than an even share)."""
    if axes == 1 or half < axes:
        return [half]
    later = [rng.randint(max(1, half // (2 * axes)), half // axes) for _ in range(axes - 1)]
    return [half - sum(later)] + later


LAYOUTS = [(28, 4, 128), (40, 8, 128), (14, 2, 64), (3, 1, 32), (8, 8, 80), (16, 2, 112), (32, 1, 64), (12, 4, 96), (6, 3, 16)]


def draw(rng):
    op = rng.choice(["rotate", "append", "shared", "shared"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if op == "rotate":
        hd = rng.choice([32, 64, 72, 80, 96, 128])
        heads = rng.choice([2, 6, 16, 24, 32])
        rows = _log(rng, 1, min(65536, ROTATE_ELEMENTS // (heads * hd * (2 if dtype == "float32" else 1))))
        rot = hd if rng.random() < 0.7 else hd // 2
        return _unnamed(rotate_case("", dtype, rows, heads, hd, _sections(rng, rot // 2, rng.choice([2, 3])),
                                    beside=rng.choice([0, heads // 2]), interleaved=rng.random() < 0.4, neighbours=rng.random() < 0.4))
    heads, kv, hd = rng.choice(LAYOUTS)
    if op == "append":
        seqs = _log(rng, 1, 24)
        budget = APPEND_ELEMENTS // ((heads + 2 * kv) * hd * (2 if dtype == "float32" else 1))
        longest = 1 if rng.random() < 0.3 else max(1, min(16000, budget // seqs))
        q_lens = [_log(rng, 1, longest) for _ in range(seqs)]
        pos0 = [rng.choice([0, rng.randint(0, 3000)]) for _ in range(seqs)]
        rot = hd if rng.random() < 0.7 else hd // 2
        return _unnamed(append_case("", dtype, q_lens, heads, kv, hd, _sections(rng, rot // 2, rng.choice([2, 3])), pos0,
                                    interleaved=rng.random() < 0.4, neighbours=rng.random() < 0.3))
    f32 = dtype == "float32"
    while True:
        seqs = _log(rng, 1, 16 if f32 else 64)
        decode = rng.random() < 0.6
        q_lens = [1] * seqs if decode else [_log(rng, 1, 24 if f32 else 256) for _ in range(seqs)]
        prefix = _log(rng, 1, 4000 if f32 else 32000)
        own_lens = [q + (_log(rng, 1, 200 if f32 else 1500) - 1 if rng.random() < 0.7 else 0) for q in q_lens]
        window = rng.choice([0, 0, 0, _log(rng, 8, 4096)])
        c = _unnamed(shared_case("", dtype, q_lens, prefix, own_lens, heads, kv, hd, window))
        w = work(c)
        scores = heads * max(sum(q_lens) * prefix, 3 * seqs * max(q_lens) * (max(own_lens) + PAGE))
        if w["flops"] <= (SHARED_FLOPS_F32 if f32 else SHARED_FLOPS) and w["bytes"] <= SHARED_BYTES and scores <= SHARED_SCORES:
            return c


def _unnamed(case):
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    case = _lists(case)
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "rotate":
        n = case["rows"] * case["heads"] * case["hd"]
        return {"bytes": 2 * n * size + 4 * case["rows"] * len(case["sections"]),
                "flops": 6 * case["rows"] * case["heads"] * sum(case["sections"])}
    rows = sum(case["q_lens"])
    if case["op"] == "append":
        n = rows * (case["heads"] + 2 * case["kv_heads"]) * case["hd"]
        return {"bytes": 2 * n * size + 4 * rows * (2 + len(case["sections"])),
                "flops": 6 * rows * (case["heads"] + case["kv_heads"]) * sum(case["sections"])}
    pairs, far = 0, case["prefix"]             # far: the first prefix key that some row sees
    kept = 0                                   # own keys that some row sees
    w = case["window"]
    for q, n in zip(case["q_lens"], case["own_lens"]):
        first = case["prefix"] + n - q         # position of the first new token
        last = case["prefix"] + n - 1
        if w <= 0 or last < w:
            pairs += sum(range(first + 1, last + 2))
        else:
            pairs += sum(min(p + 1, w) for p in range(first, last + 1))
        lo = max(0, first - w + 1) if w > 0 else 0
        far = min(far, lo)
        kept += n - max(0, lo - case["prefix"])
    keys = case["prefix"] - far + kept
    return {"bytes": size * (2 * rows * case["heads"] * case["hd"] + 2 * keys * case["kv_heads"] * case["hd"]),
            "flops": 4 * case["hd"] * case["heads"] * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _positions(n, axes, start, g):
    """Positions [n, axes] of n tokens from `start` on, as an image or a video in a text has them: runs of text (all axes the same)
    and grids (time, height, width, or height and width), the text after a grid going on from its largest position."""
    out = torch.empty((n, axes), dtype=torch.int64)
    done, at, grid = 0, start, bool(torch.randint(0, 2, (1,), generator=g))
    while done < n:
        if grid:
            w = int(torch.randint(8, 49, (1,), generator=g))
            h = int(torch.randint(8, 49, (1,), generator=g))
            left = n - done
            frames = max(1, min(64, left // (h * w))) if axes > 2 else 1
            count = min(left, frames * h * w)
            i = torch.arange(count)
            cols = [i // (h * w), i // w % h, i % w] if axes > 2 else [i // w % h, i % w]
            out[done:done + count] = at + torch.stack(cols, 1)
            at += max(frames, h, w)
        else:
            count = min(n - done, int(torch.randint(1, 40, (1,), generator=g)))
            out[done:done + count] = (at + torch.arange(count))[:, None]
            at += count
        done += count
        grid = not grid
    return out.to(torch.int32)


def _denominators(case):
    """theta^(i / half): a ladder over all pairs; patches of two axes have a ladder of their own for each axis."""
    sections, half = case["sections"], sum(case["sections"])
    if case["op"] == "rotate" and len(sections) == 2 and not case["interleaved"]:
        ladder = torch.cat([10000.0 ** (torch.arange(s, dtype=torch.float64) / s) for s in sections])
    else:
        ladder = 1000000.0 ** (torch.arange(half, dtype=torch.float64) / half)
    return ladder.float().cuda()


def _tables(g, lists):
    """Shuffled page numbers for every list's page count: (tables [n, widest] with -1 behind a list's end, pages in use and spare)."""
    counts = list(lists)
    total = sum(counts)
    perm = torch.randperm(total + 3, generator=g)
    out = torch.full((len(counts), max(max(counts), 1)), -1, dtype=torch.int64)
    at = 0
    for i, c in enumerate(counts):
        out[i, :c] = perm[at:at + c]
        at += c
    return out.to(torch.int32), total + 3


class Geometry:
    """What a step's rows are: sequence s has rows seq_start[s] .. seq_start[s] + seq_qlen[s] - 1, the first at position seq_pos0[s]."""

    def __init__(self, q_lens, pos0):
        starts = [0]
        for q in q_lens[:-1]:
            starts.append(starts[-1] + q)
        self.n_seqs, self.max_q_len = len(q_lens), max(q_lens)
        self.max_kv_len = max(q + p for q, p in zip(q_lens, pos0))
        self.decode = self.max_q_len == 1
        self.seq_start, self.seq_qlen, self.seq_pos0 = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (starts, q_lens, pos0))


class State:
    pass


def prepare(case, seed):
    case = _lists(case)
    g = torch.Generator().manual_seed(seed)
    dg = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=dg, device="cuda") * scale).to(dtype)

    s = State()
    s.case, s.hd = case, case["hd"]
    if case["op"] == "rotate":
        s.x = normal(case["rows"], (case["heads"] + case["beside"]) * case["hd"])
        s.positions = _positions(case["rows"], len(case["sections"]), 0, g).cuda()
        s.denom = _denominators(case)
        s.out = torch.empty((case["rows"], case["heads"] * case["hd"]), dtype=dtype, device="cuda")
        return s
    q_lens = case["q_lens"]
    rows = sum(q_lens)
    heads, kv, hd = case["heads"], case["kv_heads"], case["hd"]
    if case["op"] == "append":
        pos0 = case["pos0"]
        s.qkv = normal(rows, (heads + 2 * kv) * hd)
        s.positions = torch.cat([_positions(q, len(case["sections"]), max(0, p - p // 3), g) for q, p in zip(q_lens, pos0)]).cuda()
        s.denom = _denominators(case)
        table, pages = _tables(g, [(q + p + PAGE - 1) // PAGE for q, p in zip(q_lens, pos0)])
        s.q = torch.empty((rows, heads * hd), dtype=dtype, device="cuda")
    else:
        prefix = case["prefix"]
        pos0 = [prefix + n - q for q, n in zip(q_lens, case["own_lens"])]
        prefix_pages = (prefix + PAGE - 1) // PAGE
        tables, pages = _tables(g, [prefix_pages] + [(n + PAGE - 1) // PAGE for n in case["own_lens"]])
        s.prefix_table = tables[0, :prefix_pages].clone().cuda()
        table = tables[1:, :max((n + PAGE - 1) // PAGE for n in case["own_lens"])].contiguous()
        s.q = normal(rows, heads * hd, scale=1.5)
        s.out = torch.empty((rows, heads * hd), dtype=dtype, device="cuda")
    s.block_table = table.cuda()
    s.k_pool, s.v_pool = normal(pages, PAGE, kv, hd), normal(pages, PAGE, kv, hd)
    s.row_seq = torch.tensor([i for i, q in enumerate(q_lens) for _ in range(q)], dtype=torch.int32, device="cuda")
    s.row_pos = torch.tensor([p + t for q, p in zip(q_lens, pos0) for t in range(q)], dtype=torch.int32, device="cuda")
    s.geometry = Geometry(q_lens, pos0)
    s.scale = hd ** -0.5
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(s):
    c = s.case
    if own:
        return _own(s, c)
    return {"rotate": _plain_rotate, "append": _plain_append, "shared": _plain_shared}[c["op"]](s, c)


def _own(s, c):
    from friday_inference_engine_b200 import ops
    if c["op"] == "rotate":
        return ops.rotate_axes(s.x, s.positions, s.denom, c["sections"], c["heads"], s.hd, interleaved=c["interleaved"],
                               neighbours=c["neighbours"], out=s.out)
    if c["op"] == "append":
        ops.rope_axes_kv_write(s.qkv, s.row_seq, s.row_pos, s.positions, s.denom, c["sections"], c["heads"], c["kv_heads"], s.hd,
                               s.k_pool, s.v_pool, s.block_table, PAGE, interleaved=c["interleaved"], neighbours=c["neighbours"], q_out=s.q)
        return s.q, s.k_pool, s.v_pool
    ops.attention_shared(s.q, s.q.stride(0), s.out, s.k_pool, s.v_pool, s.prefix_table, c["prefix"], s.block_table, PAGE, s.row_seq,
                         s.row_pos, c["heads"], c["kv_heads"], s.hd, c["window"], s.scale, s.geometry)
    return s.out


def _axis_of(c):
    """The axis that turns each pair."""
    sections, n = c["sections"], len(c["sections"])
    if not c["interleaved"]:
        return [a for a, count in enumerate(sections) for _ in range(count)]
    return [i % n if i < n * sections[i % n] else 0 for i in range(sum(sections))]


def _plain_turn(x, positions, denom, c):
    """x [rows, heads, hd] fp32 with its first pairs turned."""
    half = sum(c["sections"])
    axis = torch.tensor(_axis_of(c), device="cuda")
    angle = positions.double()[:, axis] / denom.double()
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    if c["neighbours"]:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_rotate(s, c):
    n = c["heads"] * s.hd
    x = s.x[:, :n].float().view(c["rows"], c["heads"], s.hd)
    s.out.copy_(_plain_turn(x, s.positions, s.denom, c).view(c["rows"], n))
    return s.out


def _plain_append(s, c):
    rows, heads, kv, hd = s.qkv.shape[0], c["heads"], c["kv_heads"], s.hd
    x = s.qkv.view(rows, heads + 2 * kv, hd)
    turned = _plain_turn(x[:, :heads + kv].float(), s.positions, s.denom, c).to(x.dtype)
    s.q.copy_(turned[:, :heads].reshape(rows, heads * hd))
    page = s.block_table[s.row_seq.long(), (s.row_pos // PAGE).long()].long()
    place = (s.row_pos % PAGE).long()
    s.k_pool[page, place] = turned[:, heads:]
    s.v_pool[page, place] = x[:, heads + kv:]
    return s.q, s.k_pool, s.v_pool


def _plain_shared(s, c):
    rows, heads, kv, hd, prefix, n = s.q.shape[0], c["heads"], c["kv_heads"], s.hd, c["prefix"], len(c["q_lens"])
    group, most = heads // kv, s.geometry.max_q_len
    seq, pos = s.row_seq.long(), s.row_pos.long()
    at = torch.arange(rows, device="cuda") - s.geometry.seq_start.long()[seq]          # the row's number in its sequence
    q = s.q.float().view(rows, kv, group, hd)
    # the prefix: all rows against the same keys
    pk = s.k_pool[s.prefix_table.long()].flatten(0, 1)[:prefix].float().permute(1, 0, 2)
    pv = s.v_pool[s.prefix_table.long()].flatten(0, 1)[:prefix].float().permute(1, 0, 2)
    score_p = torch.matmul(q.permute(1, 0, 2, 3).reshape(kv, rows * group, hd), pk.transpose(1, 2)) * s.scale
    score_p = score_p.view(kv, rows, group, prefix)
    # every sequence's own keys, in whole pages, the rows of a sequence side by side
    ok = s.k_pool[s.block_table.clamp(min=0).long()].flatten(1, 2).float().permute(0, 2, 1, 3)
    ov = s.v_pool[s.block_table.clamp(min=0).long()].flatten(1, 2).float().permute(0, 2, 1, 3)
    held = ok.shape[2]
    padded = torch.zeros((n, most, kv, group, hd), device="cuda")
    padded[seq, at] = q
    score_o = torch.matmul(padded.permute(0, 2, 1, 3, 4).reshape(n, kv, most * group, hd), ok.transpose(2, 3)) * s.scale
    score_o = score_o.view(n, kv, most, group, held).permute(0, 2, 1, 3, 4)[seq, at].permute(1, 0, 2, 3)
    j = torch.arange(prefix + held, device="cuda")
    seen = j <= pos[:, None]
    if c["window"] > 0:
        seen = seen & (j > pos[:, None] - c["window"])
    score = torch.cat((score_p, score_o), -1).masked_fill(~seen[None, :, None, :], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    weight = weight / weight.sum(-1, keepdim=True)
    out = torch.matmul(weight[..., :prefix].reshape(kv, rows * group, prefix), pv).view(kv, rows, group, hd).permute(1, 0, 2, 3)
    padded_w = torch.zeros((n, most, kv, group, held), device="cuda")
    padded_w[seq, at] = weight[..., prefix:].permute(1, 0, 2, 3)
    own_out = torch.matmul(padded_w.permute(0, 2, 1, 3, 4).reshape(n, kv, most * group, held), ov)
    out = out + own_out.view(n, kv, most, group, hd).permute(0, 2, 1, 3, 4)[seq, at]
    s.out.copy_(out.reshape(rows, heads * hd))
    return s.out


# ---------------------------------------------------------------------------
# the same in 64-bit, from the definitions
# ---------------------------------------------------------------------------
def _exact_turn(x, positions, denom, c):
    """x [rows, heads, hd] double; pair by pair."""
    out, half = x.clone(), sum(c["sections"])
    bounds = [sum(c["sections"][:a + 1]) for a in range(len(c["sections"]))]
    n = len(bounds)
    for i in range(half):
        if c["interleaved"]:
            axis = i % n
            if i >= n * c["sections"][axis]:
                axis = 0
        else:
            axis = next(a for a in range(n) if i < bounds[a])
        angle = (positions[:, axis].double() / float(denom[i]))[:, None]
        first, second = (2 * i, 2 * i + 1) if c["neighbours"] else (i, i + half)
        out[:, :, first] = x[:, :, first] * angle.cos() - x[:, :, second] * angle.sin()
        out[:, :, second] = x[:, :, second] * angle.cos() + x[:, :, first] * angle.sin()
    return out


def exact(case, seed):
    s, c = prepare(case, seed), _lists(case)
    if c["op"] == "rotate":
        n = c["heads"] * s.hd
        denom = s.denom.double().cpu()
        return _exact_turn(s.x[:, :n].double().view(c["rows"], c["heads"], s.hd), s.positions, denom, c).view(c["rows"], n)
    heads, kv, hd = c["heads"], c["kv_heads"], s.hd
    if c["op"] == "append":
        x = s.qkv.double().view(-1, heads + 2 * kv, hd)
        denom = s.denom.double().cpu()
        turned = _exact_turn(x[:, :heads + kv], s.positions, denom, c)
        k_pool, v_pool = s.k_pool.double(), s.v_pool.double()
        row = 0
        for i, (q, p) in enumerate(zip(c["q_lens"], c["pos0"])):
            places = torch.arange(p, p + q, device="cuda")
            flat = s.block_table[i].long()[places // PAGE] * PAGE + places % PAGE
            k_pool.view(-1, kv, hd)[flat] = turned[row:row + q, heads:]
            v_pool.view(-1, kv, hd)[flat] = x[row:row + q, heads + kv:]
            row += q
        return turned[:, :heads].reshape(-1, heads * hd), k_pool, v_pool
    out = torch.zeros((s.q.shape[0], heads, hd), dtype=torch.float64, device="cuda")
    row = 0
    for i, (q, n) in enumerate(zip(c["q_lens"], c["own_lens"])):
        own_pages = s.block_table[i, :(n + PAGE - 1) // PAGE].long()
        keys = torch.cat((s.k_pool[s.prefix_table.long()].flatten(0, 1)[:c["prefix"]], s.k_pool[own_pages].flatten(0, 1)[:n])).double()
        values = torch.cat((s.v_pool[s.prefix_table.long()].flatten(0, 1)[:c["prefix"]], s.v_pool[own_pages].flatten(0, 1)[:n])).double()
        place = torch.arange(keys.shape[0], device="cuda")
        pos = torch.arange(c["prefix"] + n - q, c["prefix"] + n, device="cuda")[:, None]
        seen = (place <= pos) & ((place > pos - c["window"]) if c["window"] > 0 else True)
        queries = s.q[row:row + q].double().view(q, heads, hd)
        for h in range(heads):
            score = queries[:, h] @ keys[:, h // (heads // kv)].T * hd ** -0.5
            p = torch.softmax(score.masked_fill(~seen, -math.inf), -1)
            out[row:row + q, h] = p @ values[:, h // (heads // kv)]
        row += q
    return out.view(-1, heads * hd)
