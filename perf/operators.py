"""The operators of the paged 4-bit K/V cache, as they are measured: appending keys and values (position rotation,
quantisation to 4 bits), reading entries back, and attention over the cache.

A case is a dict of plain values; ``run`` makes one pass through an operator in its plain form (elementary torch
operations in 32 bits) or, where ``own`` is true, through this framework's kernels.

The quantiser.  A 64-value vector x of norm n is rotated, y = H (signs * x[perm]) with the Walsh-Hadamard matrix H (no
1/8), and coordinate i is held as a sign and the number of bounds b_j with |y_i| > b_j * 8n; the norm is held in 16 bits.
It stands for x[perm[i]] = signs_i * (H c)_i * n / 8 with c the codes' levels.  Sums of squares are added in halves
(32 + 32, 16 + 16, ...), so that the same codes come out wherever it runs.
"""

import math

import torch

own = False

D = 64
THETA = 10000.0
# Lloyd-Max levels and bounds of one coordinate of a uniform point on the 64-sphere, 16 levels, upper half (the lower is
# its mirror image).
LEVELS = (0.0157579668, 0.0476557687, 0.0806962475, 0.115755357, 0.154124632, 0.198039144, 0.252138406, 0.330133021)
BOUNDS = (0.0317068696, 0.0641760081, 0.0982258022, 0.134939998, 0.176081896, 0.225088775, 0.291135699)
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
NORMS = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------- cases --
def listed():
    return [
        # one new token of each of 48 running sequences (one left idle): the append of a serving step, where latency counts
        dict(name="append_step", op="append", seqs=48, heads=12, page=64, dtype="bf16", norm="f16", new=1, context=4096,
             ragged=True, idle=1, masked=0),
        # the encoder's whole batch: 256 series of 133 tokens (context 2048: 128 patches, the register token, 4 to
        # forecast), 12 heads, some patches missing
        dict(name="append_series", op="append", seqs=256, heads=12, page=64, dtype="bf16", norm="f16", new=133, context=133,
             ragged=False, idle=0, masked=20),
        # fp32 model, ragged chunks, small pages, an odd head count: everything that is not a multiple of anything
        dict(name="append_ragged_f32", op="append", seqs=7, heads=3, page=16, dtype="f32", norm="bf16", new=1531, context=2777,
             ragged=True, idle=1, masked=50),
        # a long prompt taken in at once, grouped heads
        dict(name="append_long", op="append", seqs=2, heads=8, page=128, dtype="bf16", norm="f16", new=65536, context=65536,
             ragged=False, idle=0, masked=0),
        # the entries of one short series brought back
        dict(name="read_series", op="read", seqs=1, heads=12, page=64, dtype="bf16", norm="f16", new=133, context=133,
             ragged=False, idle=0, masked=0),
        # a batch of long sequences moved out of the cache
        dict(name="read_batch", op="read", seqs=24, heads=8, page=32, dtype="f32", norm="f16", new=4001, context=8192,
             ragged=True, idle=0, masked=0),
        # one query token over one encoded series of 133 tokens: the smallest step
        dict(name="attend_token_short", op="attend", seqs=1, heads=12, group=1, page=64, dtype="bf16", norm="f16", new=1,
             context=133, ragged=False, idle=0, masked=0, causal=True, rotate=True),
        # a serving step: 64 sequences of up to 16384 tokens (one idle), a head of keys for each of the 12 query heads
        dict(name="attend_step_batch", op="attend", seqs=64, heads=12, group=1, page=64, dtype="bf16", norm="f16", new=1,
             context=16384, ragged=True, idle=1, masked=10, causal=True, rotate=True),
        # one very long sequence, four query heads to a head of keys: the long axis has to be split
        dict(name="attend_step_long", op="attend", seqs=1, heads=8, group=4, page=64, dtype="bf16", norm="f16", new=1,
             context=131071, ragged=False, idle=0, masked=0, causal=True, rotate=True),
        # a few tokens at a time in fp32, with log-sum-exp for joining with other keys; small pages, odd sizes, masks
        dict(name="attend_few_f32", op="attend", seqs=5, heads=3, group=2, page=16, dtype="f32", norm="bf16", new=5,
             context=2777, ragged=True, idle=1, masked=50, causal=True, rotate=True),
        # the encoder's attention over its cached batch: 256 series, all 133 tokens see all, masked patches
        dict(name="attend_series", op="attend", seqs=256, heads=12, group=1, page=64, dtype="bf16", norm="f16", new=133,
             context=133, ragged=False, idle=0, masked=20, causal=False, rotate=True),
        # chunks of long prompts, causal, grouped heads, ragged
        dict(name="attend_chunk", op="attend", seqs=3, heads=8, group=4, page=128, dtype="bf16", norm="f16", new=2048,
             context=16384, ragged=True, idle=0, masked=0, causal=True, rotate=True),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    case = dict(op=rng.choice(("append", "read", "attend", "attend")), heads=rng.choice((1, 2, 3, 5, 8, 12)),
                page=rng.choice((16, 32, 64, 128)), dtype=rng.choice(("bf16", "bf16", "f32")),
                norm=rng.choice(("f16", "bf16")), ragged=rng.random() < 0.6, masked=rng.choice((0, 0, 10, 100)))
    if case["op"] == "attend":
        case["group"] = rng.choice((1, 1, 2, 3, 4, 8))
        case["causal"], case["rotate"] = rng.random() < 0.7, rng.random() < 0.8
        kind = rng.choice(("step", "few", "chunk"))
        if kind == "chunk":
            case["dtype"] = "bf16"  # an fp32 prompt chunk is a check of the model's numerics, not a load
            case["new"], most = _log(rng, 17, 2048), 2 << 30  # rows x keys, over all query heads
        else:
            case["new"], most = 1 if kind == "step" else rng.randint(2, 9), 3 << 28
        case["context"] = _log(rng, max(case["new"], 16), 131072 if kind == "step" else max(16384, case["new"]))
        each = case["new"] * case["context"] * case["heads"] * case["group"]
        room = min(most // each, (1 << 20) // (case["context"] * case["heads"] // 8 + 1))
        case["seqs"] = _log(rng, 1, max(1, min(256, room)))
        if room < 1:
            case["heads"], case["group"] = 1, 1
    else:
        case["new"] = _log(rng, 1, 65536)
        case["context"] = case["new"] + _log(rng, 1, 8192) - 1
        case["seqs"] = _log(rng, 1, max(1, min(256, (1 << 20) // (case["new"] * case["heads"]))))
    case["idle"] = rng.randint(0, 1) if case["seqs"] > 1 else 0
    return case


def _lengths(case):
    """-> (tokens in each sequence's cache, its new or asked-for tokens).  Where the case is ragged the lengths fall from
    the longest to about an eighth of it; idle sequences have no token in the cache."""
    n, at = case["seqs"], []
    for i in range(n):
        f = 1.0 if not case["ragged"] or i == 0 else 1.0 - 0.875 * i / n
        new = max(1, int(case["new"] * f))
        at.append((max(new, int(case["context"] * f) - (i * 7919) % 13 * (1 if f < 1 else 0)), new))
    for i in range(case["idle"]):
        at[n - 1 - i] = (0, at[n - 1 - i][1] if case["op"] == "attend" else 0)
    return at


def work(case):
    at, h, e = _lengths(case), case["heads"], 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("append", "read"):
        t = sum(n for _, n in at)
        # append: k and v in, entries out, and the values they stand for, which the pass gives back; read: entries in, values out
        by = t * h * (2 * D * e + 68 + (0 if case["op"] == "read" else 2 * D * e))
        return {"bytes": by, "flops": t * h * 2 * 6 * D * (2 if case["op"] == "append" else 1)}
    qh = h * case["group"]
    by = sum(c * h * 68 + n * qh * D * 2 * e for c, n in at)
    pairs = sum(n * c - (n * (n - 1) // 2 if case["causal"] and c >= n else 0) for c, n in at)
    return {"bytes": by, "flops": 4.0 * D * pairs * qh}


# --------------------------------------------------------------------------- inputs --
def _rope_table(rows):
    inv = 1.0 / THETA ** (torch.arange(0, D, 2, dtype=torch.int64).float() / D)
    ang = torch.arange(rows, dtype=torch.float32, device="cuda")[:, None] * inv.cuda()[None]
    return torch.stack([ang.double().cos(), ang.double().sin()], -1).float()


def _rotation(seed):
    """Random signs and permutation of one quantiser (host generator)."""
    g = torch.Generator().manual_seed(seed)
    signs = torch.where(torch.rand(D, generator=g) > 0.5, 1.0, -1.0)
    return signs, torch.randperm(D, generator=g)


def _data(case, seed):
    """k, v (all tokens, heads, 64) with each token's sequence, position and mask, q, lengths, page table.  Keys have the
    shape that models give them: a few channels much larger than the rest, and an offset that all tokens share."""
    g = torch.Generator("cuda").manual_seed(seed)
    at, h, dt = _lengths(case), case["heads"], DTYPES[case["dtype"]]
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    have = torch.tensor([c for c, _ in at], dtype=torch.int32, device="cuda")
    new = torch.tensor([n for _, n in at], dtype=torch.int32, device="cuda")
    stored = have if case["op"] == "attend" else new  # tokens of each sequence that are quantised
    first = have - stored
    seq = torch.repeat_interleave(torch.arange(len(at), device="cuda"), stored.long()).int()
    ends = torch.cumsum(stored, 0)
    pos = (torch.arange(len(seq), device="cuda") - (ends - stored)[seq.long()] + first[seq.long()]).int()
    wide = torch.exp(0.5 * normal(1, h, D))
    k = (normal(len(seq), h, D) * wide + normal(1, h, D)).to(dt)
    v = (normal(len(seq), h, D) * torch.exp(0.5 * normal(len(seq), h, 1))).to(dt)
    mask = None
    if case["masked"]:
        mask = torch.rand(len(seq), generator=g, device="cuda") >= case["masked"] / 1000
        mask = mask.to(torch.uint8)
    wide_pages = -(-max(max(c for c, _ in at), 1) // case["page"])
    pages = len(at) * wide_pages
    table = torch.randperm(pages, generator=g, device="cuda").view(len(at), wide_pages).int()
    q = cu = None
    if case["op"] == "attend":
        cu = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int32), torch.cumsum(new, 0).int()])
        q = (normal(sum(n for _, n in at), h * case["group"], D) * 1.2).to(dt)
    return dict(k=k, v=v, seq=seq, pos=pos, mask=mask, table=table, pages=pages, q=q, cu=cu, have=have,
                seeds=(seed % 100003, seed % 100003 + 1))


def prepare(case, seed):
    d = _data(case, seed)
    at = _lengths(case)
    rows = max(max(c for c, _ in at), 1)
    d.update(case=case, longest=rows, most_new=max(n for _, n in at), scale=0.125)
    if own:
        from cutechronos_b200.kvcache import PagedKV4Cache
        from cutechronos_b200.turboquant import TurboQuantParams

        norm = {"f16": "float16", "bf16": "bfloat16"}[case["norm"]]
        key, value = (TurboQuantParams.build(D, 4, mode="mse", seed=s, norm_dtype=norm, device="cuda") for s in d["seeds"])
        d["cache"] = PagedKV4Cache(d["pages"], case["heads"], page_size=case["page"], key=key, value=value,
                                   rope_theta=THETA, max_positions=rows, device="cuda")
        if case["op"] != "append":
            d["cache"].append(d["k"], d["v"], d["seq"], d["pos"], d["table"], token_mask=d["mask"])
    else:
        d["rope"] = _rope_table(rows)
        d["levels"] = torch.tensor([*LEVELS, *(-x for x in LEVELS)], device="cuda")
        d["bounds"] = torch.tensor(BOUNDS, device="cuda")
        d["rot"] = [(s.cuda(), p.cuda()) for s, p in map(_rotation, d["seeds"])]
        shape = (d["pages"], case["page"], case["heads"])
        d["codes"] = [torch.zeros(*shape, D, dtype=torch.uint8, device="cuda") for _ in range(2)]
        d["norms"] = [torch.zeros(*shape, dtype=NORMS[case["norm"]], device="cuda") for _ in range(2)]
        d["seen"] = torch.zeros(*shape[:2], dtype=torch.bool, device="cuda")
        if case["op"] != "append":
            for i in range(0, len(d["seq"]), 1 << 16):  # in parts: the plain quantiser's temporaries are large
                _append(d, slice(i, i + (1 << 16)))
    if case["op"] != "append":
        del d["k"], d["v"]
    if case["op"] == "attend":
        del d["seq"], d["pos"], d["mask"]
    return d


# ----------------------------------------------------------------------- plain forms --
def _hadamard(y):
    """Walsh-Hadamard butterflies of width 1, 2, ..., 32 over the last axis."""
    s = y.shape
    w = 1
    while w < D:
        y = y.reshape(*s[:-1], D // (2 * w), 2, w)
        y = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], -2).reshape(s)
        w *= 2
    return y


def _turn(x, cs):
    """Rotates the halves (x[i], x[i + 32]) by the position's angles; cs (..., 32, 2)."""
    a, b, c, s = x[..., : D // 2], x[..., D // 2:], cs[..., 0], cs[..., 1]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _quantise(x, rot, bounds, norm_type):
    signs, perm = rot
    y = _hadamard(x[..., perm] * signs)
    s = x * x
    w = D // 2
    while w:
        s = s[..., :w] + s[..., w:2 * w]
        w //= 2
    n = s[..., 0].sqrt()
    over = (y.abs()[..., None] > (bounds * (8 * n[..., None]))[..., None, :]).sum(-1)
    held = torch.where(n.isfinite(), n.clamp(max=65504.0), torch.nan).to(norm_type)
    return (over + 8 * (y < 0)).to(torch.uint8), held


def _append(d, part=slice(None)):
    seq, pos = d["seq"][part].long(), d["pos"][part].long()
    page = d["case"]["page"]
    at = (d["table"][seq, pos // page].long(), pos % page)
    x = (_turn(d["k"][part].float(), d["rope"][pos][:, None]), d["v"][part].float())
    for i in range(2):
        codes, norms = _quantise(x[i], d["rot"][i], d["bounds"], d["norms"][i].dtype)
        d["codes"][i].index_put_(at, codes)
        d["norms"][i].index_put_(at, norms)
    d["seen"].index_put_(at, torch.ones_like(pos, dtype=torch.bool) if d["mask"] is None else d["mask"][part].bool())


def _read(d):
    seq, pos = d["seq"].long(), d["pos"].long()
    page = d["case"]["page"]
    at = (d["table"][seq, pos // page].long(), pos % page)
    out = []
    for i in range(2):
        signs, perm = d["rot"][i]
        z = _hadamard(d["levels"][d["codes"][i][at].long()]) * (d["norms"][i][at].float() * 0.125)[..., None] * signs
        out.append(z[..., perm.argsort()].to(DTYPES[d["case"]["dtype"]]))
    return out


def _attend(d):
    case = d["case"]
    b, h, g = case["seqs"], case["heads"], case["group"]
    dt, dev = DTYPES[case["dtype"]], d["q"].device
    n, length = d["most_new"], d["table"].shape[1] * case["page"]
    kv = []
    for i in range(2):
        signs, perm = d["rot"][i]
        back = (_hadamard(torch.eye(D, device=dev)) * 0.125 * signs)[:, perm.argsort()]
        c = d["levels"][d["codes"][i][d["table"].long()].view(b, length, h, D).int()]
        x = c * d["norms"][i][d["table"].long()].float().view(b, length, h, 1)
        kv.append((x @ back).transpose(1, 2))
    # queries in a frame of equal lengths (the last row of a sequence stands at its last cached token)
    new = d["cu"][1:] - d["cu"][:-1]
    rows = torch.arange(n, device=dev)
    real = rows < new[:, None]
    where = (d["cu"][:-1, None] + rows).clamp(max=len(d["q"]) - 1).long()
    q = d["q"][where].float()
    last = d["have"][:, None] - new[:, None] + rows  # each row's own position
    if case["rotate"]:
        q = _turn(q, d["rope"][last.clamp(0, d["longest"] - 1).long()][:, :, None])
    q = q.view(b, n, h, g, D).permute(0, 2, 3, 1, 4).reshape(b, h, g * n, D)
    keys = torch.arange(length, device=dev)
    seen = (keys < d["have"][:, None]) & d["seen"][d["table"].long()].view(b, length)
    seen = seen[:, None, :] & ((keys <= last[:, :, None]) if case["causal"] else torch.ones_like(keys, dtype=torch.bool))
    s = (q @ kv[0].transpose(2, 3)).mul_(d["scale"]).view(b, h, g, n, length)
    s.masked_fill_(~seen[:, None, None], -torch.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -torch.inf, 0.0, m)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where(seen.any(1)[:, None, :, None], kv[1], 0.0)
    o = (p.view(b, h, g * n, length) @ v).view(b, h, g, n, D) / torch.where(total == 0, 1.0, total)
    lse = (m + total.log()).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, n, h * g, D)[real].to(dt)
    if case["dtype"] == "f32":
        return [o, lse.permute(0, 3, 1, 2).reshape(b, n, h * g)[real]]
    return [o]


def run(d):
    case = d["case"]
    if not own:
        if case["op"] == "attend":
            return _attend(d)
        if case["op"] == "append":
            _append(d)
        return _read(d)
    cache = d["cache"]
    if case["op"] == "attend":
        f32 = case["dtype"] == "f32"  # where the caller joins with other keys: log-sum-exp too
        out = cache.attention(d["q"], d["have"], d["table"], cu_q=d["cu"], max_q=d["most_new"], max_len=d["longest"],
                              causal=case["causal"], scale=d["scale"], rotate_q=case["rotate"], return_lse=f32)
        return list(out) if f32 else [out]
    if case["op"] == "append":
        cache.append(d["k"], d["v"], d["seq"], d["pos"], d["table"], token_mask=d["mask"])
    return list(cache.read(d["seq"], d["pos"], d["table"], dtype=DTYPES[case["dtype"]]))


# ------------------------------------------------------------------------ in 64 bits --
def _held(x, rot, norm_type):
    """What the cache stands for after x (float64) is put in, rotated: nearest level of each coordinate of the unit
    vector, times the norm as it is held."""
    signs, perm = (t.cuda() for t in rot)
    n = x.square().sum(-1, keepdim=True).sqrt()
    y = ((x / n)[..., perm] * signs) @ _walsh()
    lv = torch.tensor(sorted([*LEVELS, *(-v for v in LEVELS)]), device="cuda").double()
    up = torch.tensor(BOUNDS, device="cuda").double()
    cuts = torch.cat([-up.flip(0), torch.zeros(1, device="cuda", dtype=torch.float64), up])
    c = lv[torch.bucketize(y, cuts)]
    back = ((c @ _walsh()) * signs)[..., perm.argsort()]
    return back * n.clamp(max=65504.0).to(norm_type).double()


def _walsh():
    i = torch.arange(D)
    bits = (i[:, None] & i)[..., None] >> torch.arange(6) & 1
    return (1 - 2 * (bits.sum(-1) % 2)).double().cuda() / 8


def exact(case, seed):
    d = _data(case, seed)
    at, h = _lengths(case), case["heads"]
    rope = _rope_table(max(max(c for c, _ in at), 1)).double()
    rot = [_rotation(s) for s in d["seeds"]]
    norm = NORMS[case["norm"]]
    if case["op"] != "attend":
        out = [torch.empty(d["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2)]
        for i in range(0, len(d["seq"]), 1 << 15):
            p = slice(i, i + (1 << 15))
            out[0][p] = _held(_turn(d["k"][p].double(), rope[d["pos"][p].long()][:, None]), rot[0], norm)
            out[1][p] = _held(d["v"][p].double(), rot[1], norm)
        return out
    g = case["group"]
    o = torch.zeros(d["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(d["q"].shape[:2], -torch.inf, dtype=torch.float64, device="cuda")
    row = key = 0
    for have, new in at:
        if have:
            part = slice(key, key + have)
            last = torch.arange(have - new, have, device="cuda")
            for i in range(h):
                kk = _held(_turn(d["k"][part, i].double(), rope[:have]), rot[0], norm)
                vv = _held(d["v"][part, i].double(), rot[1], norm)
                q = d["q"][row:row + new, i * g:(i + 1) * g].double()
                if case["rotate"]:
                    q = _turn(q, rope[last][:, None])
                s = (q.reshape(-1, D) @ kk.T).view(new, g, have) * 0.125
                if case["causal"]:
                    s.masked_fill_((torch.arange(have, device="cuda") > last[:, None])[:, None], -torch.inf)
                if d["mask"] is not None:
                    s.masked_fill_(d["mask"][part] == 0, -torch.inf)
                t = s.logsumexp(-1)
                w = torch.where(t[..., None] == -torch.inf, 0.0, (s - t[..., None]).exp())
                o[row:row + new, i * g:(i + 1) * g] = (w.view(-1, have) @ vv).view(new, g, D)
                lse[row:row + new, i * g:(i + 1) * g] = t
        row, key = row + new, key + have
    return [o, lse] if case["dtype"] == "f32" else [o]
