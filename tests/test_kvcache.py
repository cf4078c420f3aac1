"""The paged 4-bit K/V cache (append, read, attention) against plain implementations in 64 bits.

The oracle reads the cache's bytes itself: codes and norms are taken from the pages by the documented layout, so what
attention and read make of them is tested apart from what append put there.  Append is tested code by code: a code may
differ from the 64-bit decision only where the coordinate lies within fp32's error of a bound."""

from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from cutechronos_b200 import _native as nat
from cutechronos_b200.turboquant import TurboQuantParams

D = 64


# ------------------------------------------------------------------------------- oracle --
def walsh() -> torch.Tensor:
    i = torch.arange(D)
    bits = (i[:, None] & i)[..., None] >> torch.arange(6) & 1
    return (1 - 2 * (bits.sum(-1) % 2)).double()


def tables(p: TurboQuantParams):
    """levels (8), bounds (7), signs, perm in 64 bits, as the cache takes them from the quantiser."""
    cb, cut = p.tensors["codebook"].cpu(), p.tensors["boundaries"].cpu()
    return ((cb[8:] - cb[:8].flip(0)) * 0.5).double(), ((cut[8:] - cut[:7].flip(0)) * 0.5).double(), \
        p.tensors["signs"].cpu().double(), p.tensors["perm"].cpu().long()


def unpack(cache, which: int):
    """-> magnitudes (pages, page_size, heads, 64), signs (+-1), norms (float64), masked: read from the pages' bytes."""
    h, ps = cache.num_heads, cache.page_size
    b = cache.pages.cpu().view(cache.num_pages, h, ps // 16, 1088)
    codes = b[..., 512 * which:512 * which + 512].reshape(cache.num_pages, h, ps, 8, 4).long()
    word = codes[..., 0] | codes[..., 1] << 8 | codes[..., 2] << 16 | codes[..., 3] << 24
    at = torch.arange(8)
    mag = (word[..., None] >> (4 * at)) & 7
    sign = 1 - 2 * ((word[..., None] >> (4 * at + 3)) & 1)
    raw = b[..., 1024:].reshape(cache.num_pages, h, ps, 2, 2)[..., which, :].contiguous().view(torch.int16).squeeze(-1)
    kind = torch.bfloat16 if cache._c.norm_dtype else torch.float16
    norm = (raw & 0x7FFF).view(kind).double()
    flat = lambda t: t.reshape(cache.num_pages, h, ps, D).transpose(1, 2)  # noqa: E731
    return flat(mag), flat(sign), norm.transpose(1, 2), (raw < 0).transpose(1, 2)


def stands_for(cache, params, which: int):
    """The vectors the pages stand for, float64 (pages, page_size, heads, 64)."""
    mag, sign, norm, masked = unpack(cache, which)
    lv, _, signs, perm = tables(params)
    y = (lv[mag] * sign) @ walsh() * signs / 8 * norm[..., None]
    out = torch.empty_like(y)
    out[..., perm] = y
    return out, masked


def turn(x, pos, theta=10000.0):
    """Rotates the halves of x (tokens, heads, 64) in 64 bits by the fp32 angles of the positions."""
    inv = 1.0 / theta ** (torch.arange(0, D, 2, dtype=torch.int64).float() / D)
    ang = (pos.float()[:, None] * inv[None]).double()
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = x[..., :32], x[..., 32:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def oracle_attention(cache, params, q, lens, table, cu, causal, scale, rotate):
    """Returns out, lse and, for each row and head, a bound on what rounding may do (see ``allowed``)."""
    kx, masked = stands_for(cache, params[0], 0)
    vx, _ = stands_for(cache, params[1], 1)
    ps, g = cache.page_size, q.shape[1] // cache.num_heads
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    sway = torch.zeros(q.shape[:2], dtype=torch.float64)   # sum |q||K^| of the worst key, in the codes' frame
    weight = torch.zeros(q.shape[:2], dtype=torch.float64)  # sum p ||V^||
    for s, n in enumerate(lens):
        r0, r1 = cu[s], cu[s + 1]
        if r1 == r0:
            continue
        at = torch.arange(n)
        pg = table[s][at // ps].long()
        k, v, hide = kx[pg, at % ps], vx[pg, at % ps], masked[pg, at % ps]
        last = n - (r1 - r0) + torch.arange(r1 - r0)
        rows = q[r0:r1].double()
        if rotate:
            rows = turn(rows, last.clamp(min=0))
        for h in range(q.shape[1]):
            see = ~hide[:, h // g][None].expand(r1 - r0, n).clone()
            if causal:
                see &= at[None] <= last[:, None]
            x = (rows[:, h] @ k[:, h // g].T * scale).masked_fill(~see, -math.inf)
            z = x.logsumexp(-1) if n else torch.full((r1 - r0,), -math.inf, dtype=torch.float64)
            p = torch.where(see & (z[:, None] > -math.inf), (x - z[:, None]).exp(), 0.0)
            out[r0:r1, h] = torch.where(p[..., None] > 0, p[..., None] * v[None, :, h // g], 0.0).sum(1)
            lse[r0:r1, h] = z
            if n:
                # |q| . |c| n <= ||q|| ||K^||: a bound on any product's sum of magnitudes, whatever the frame
                size = abs(scale) * rows[:, h].norm(dim=-1)[:, None] * k[:, h // g].norm(dim=-1)[None]
                sway[r0:r1, h] = size.masked_fill(~see, 0.0).amax(-1)
                weight[r0:r1, h] = torch.where(p > 0, p * v[:, h // g].norm(dim=-1)[None], 0.0).sum(-1)
    return out, lse, sway, weight


def allowed(out, sway, weight, f32: bool):
    """How far a row (2-norm) and its log-sum-exp may be off.  A product of relative roundings e of q and of the levels
    moves a score by at most 2 e sum|q||K^|, hence every weight by that factor twice (numerator and sum), and the sum
    over V^ by e twice more (weight and level) next to it; the output's own rounding is 2^-9 (bf16, a row's 2-norm).  e = 2^-11
    for fp16 operands; 2^-18 for fp32 calls: two fp16 parts leave 2^-22, fp32 sums of up to 64 terms 2^-18."""
    e = 2.0 ** -18 if f32 else 2.0 ** -11
    score = 2 * e * sway + e
    return weight * (2 * score + 2 * e) + out.norm(dim=-1) * (0 if f32 else 2.0 ** -9) + 1e-30, score + 4 * e


# ------------------------------------------------------------------------------ helpers --
def make(pages, heads, page_size=64, norm="float16", theta=10000.0, max_positions=4096, seed=3):
    from cutechronos_b200.kvcache import PagedKV4Cache
    kp = TurboQuantParams.build(D, 4, mode="mse", seed=seed, norm_dtype=norm, device="cpu")
    vp = TurboQuantParams.build(D, 4, mode="mse", seed=seed + 1, norm_dtype=norm, device="cpu")
    return PagedKV4Cache(pages, heads, page_size=page_size, key=kp, value=vp, rope_theta=theta,
                         max_positions=max_positions), (kp, vp)


def filled(lens, heads, page_size=64, norm="float16", dtype=torch.bfloat16, seed=0, mask_every=0, spare=1, theta=10000.0):
    """A cache whose sequences hold ``lens`` random tokens, pages in random order -> cache, quantisers, table, k, v."""
    g = torch.Generator().manual_seed(seed)
    wide = max(1, -(-max(lens) // page_size))
    cache, params = make(len(lens) * wide + spare, heads, page_size, norm, theta)
    cache.pages.fill_(0xFF)  # unused places: NaN norms, masked: must never matter
    table = torch.randperm(len(lens) * wide + spare, generator=g)[:len(lens) * wide].view(len(lens), wide).int()
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)]).int()
    pos = torch.cat([torch.arange(n) for n in lens]).int()
    k = (torch.randn(len(seq), heads, D, generator=g) * torch.exp(torch.randn(1, heads, D, generator=g) * 0.5)).to(dtype)
    v = (torch.randn(len(seq), heads, D, generator=g) * torch.exp(torch.randn(len(seq), heads, 1, generator=g))).to(dtype)
    mask = (torch.arange(len(seq)) % mask_every != 1).to(torch.uint8) if mask_every else None
    cache.append(k.cuda(), v.cuda(), seq.cuda(), pos.cuda(), table.cuda(),
                 token_mask=mask.cuda() if mask is not None else None)
    return cache, params, table, (k, v, seq, pos, mask)


def check_codes(cache, params, table, k, v, seq, pos, theta=10000.0):
    """Every code of the tokens against the 64-bit decision."""
    ps = cache.page_size
    pg, off = table[seq.long(), pos.long() // ps].long(), pos.long() % ps
    for which, x in ((0, turn(k.double(), pos, theta) if theta else k.double()), (1, v.double())):
        mag, sign, norm, _ = unpack(cache, which)
        mag, sign, norm = mag[pg, off], sign[pg, off], norm[pg, off]
        _, bounds, signs, perm = tables(params[which])
        n = x.norm(dim=-1)
        y = (x[..., perm] * signs) @ walsh() / (8 * n).clamp(min=1e-300)[..., None]
        want = (y.abs()[..., None] > bounds).sum(-1)
        # fp32: rotation, squares, six adds of the butterflies, scaled bounds: under 2^-20 of 8n
        edge = torch.cat([bounds, torch.zeros(1, dtype=torch.float64)])
        near = (y.abs()[..., None] - edge).abs().amin(-1) < 2.0 ** -20
        live = (n > 0)[..., None] & ~near
        assert torch.equal(mag[live], want[live])
        assert torch.equal(sign[live], torch.where(y < 0, -1, 1)[live])
        assert near.double().mean() < 1e-3
        bits = 2.0 ** -8 if cache._c.norm_dtype else 2.0 ** -11  # half a spacing of the norm's type, at most
        assert ((norm - n).abs() <= n * bits * 1.01 + 2.0 ** -25).all()


# ------------------------------------------------------------------------------ CPU part --
def test_page_bytes_and_refusals_without_a_gpu():
    lib = nat.load()
    n = C.c_size_t()
    assert lib.cc2_kv4_page_bytes(64, 12, C.byref(n)) == 0 and n.value == 12 * 4 * 1088
    for bad in (0, 8, 24, 512, -16):
        assert lib.cc2_kv4_page_bytes(bad, 12, C.byref(n)) == -1 and b"page_size" in lib.cc2_last_error()
    assert lib.cc2_kv4_page_bytes(64, 0, C.byref(n)) == -1
    assert lib.cc2_kv4_append(None, 1, None, 0, 0, None, 0, 0, 1, None, None, None, None, 1, 1, None) == -1
    assert b"null cache" in lib.cc2_last_error()
    c = nat.KV4Cache(pages=1 << 20, num_pages=4, page_size=64, heads=2)
    r = C.byref(c)
    assert lib.cc2_kv4_append(r, 7, None, 0, 0, None, 0, 0, 1, None, None, None, None, 1, 1, None) == -1
    assert b"dtype" in lib.cc2_last_error()
    assert lib.cc2_kv4_append(r, 1, 1 << 20, 128, 64, 1 << 20, 128, 64, 1, None, None, None, None, 1, 1, None) == -1
    assert lib.cc2_kv4_append(r, 1, (1 << 20) + 2, 128, 64, 1 << 20, 128, 64, 1, 64, 64, None, 64, 1, 1, None) == -1
    assert b"16 bytes" in lib.cc2_last_error()
    assert lib.cc2_kv4_attention_workspace_bytes(r, 1, 3, 1, 1, 1, 64, C.byref(n)) == -1
    assert b"no multiple" in lib.cc2_last_error()
    c.norm_dtype = 2
    assert lib.cc2_kv4_read(r, 1, None, None, 1, None, None, None, 1, 1, None) == -1
    assert b"norm_dtype" in lib.cc2_last_error()


def test_cache_refuses_other_quantisers():
    from cutechronos_b200.kvcache import PagedKV4Cache
    b = lambda **kw: TurboQuantParams.build(D, kw.pop("bits", 4), device="cpu", **kw)  # noqa: E731
    for bad in (b(mode="prod"), b(bits=3), b(rotation="qr")):
        with pytest.raises(ValueError, match="quantiser must be"):
            PagedKV4Cache(4, 2, key=bad)
    with pytest.raises(ValueError, match="16 bits"):
        PagedKV4Cache(4, 2, key=b(norm_dtype="float32"), value=b(norm_dtype="float32"))
    with pytest.raises(ValueError, match="same type"):
        PagedKV4Cache(4, 2, key=b(norm_dtype="bfloat16"))
    skew = b()
    skew.tensors["codebook"] = skew.tensors["codebook"] + 0.01
    with pytest.raises(ValueError, match="symmetric"):
        PagedKV4Cache(4, 2, key=skew)
    wide = b()
    wide.tensors["codebook"], wide.tensors["boundaries"] = wide.tensors["codebook"] * 1.5, wide.tensors["boundaries"] * 1.5
    with pytest.raises(ValueError, match="share one codebook"):
        PagedKV4Cache(4, 2, key=wide)
    with pytest.raises(ValueError, match="page_size"):
        PagedKV4Cache(4, 2, page_size=48)
    with pytest.raises(ValueError, match="num_pages"):
        PagedKV4Cache(0, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        PagedKV4Cache(4, 2, device="cpu")


# ---------------------------------------------------------------------------------- append --
@pytest.mark.gpu
@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype,norm,heads", [(torch.bfloat16, "float16", 12), (torch.float32, "bfloat16", 3),
                                              (torch.float32, "float16", 1)])
def test_append_codes(page_size, dtype, norm, heads):
    cache, params, table, (k, v, seq, pos, _) = filled([0, 1, 15, 16, 17, 133, 300], heads, page_size, norm, dtype)
    check_codes(cache, params, table, k, v, seq, pos)
    cache.check()


@pytest.mark.gpu
def test_append_in_parts_gives_the_same_bytes():
    whole, params, table, (k, v, seq, pos, _) = filled([40, 133], 5)
    part, _ = make(whole.num_pages, 5)
    part.pages.fill_(0xFF)
    d = [t.cuda() for t in (k, v, seq, pos, table)]
    order = torch.randperm(len(seq), generator=torch.Generator().manual_seed(1)).cuda()
    for i in range(0, len(seq), 7):
        j = order[i:i + 7]
        part.append(d[0][j], d[1][j], d[2][j], d[3][j], d[4])
    assert torch.equal(whole.pages, part.pages)


@pytest.mark.gpu
def test_append_without_rotation_strides_and_alignment():
    g = torch.Generator().manual_seed(5)
    cache, params = make(8, 3, 32, theta=None)
    packed = torch.randn(77, 3 * 3 * D, generator=g).to(torch.bfloat16).cuda()  # [Q|K|V] rows
    k, v = packed[:, 192:384].view(77, 3, D), packed[:, 384:].view(77, 3, D)
    seq, pos = torch.zeros(77, dtype=torch.int32), torch.arange(77, dtype=torch.int32)
    table = torch.tensor([[5, 0, 3]], dtype=torch.int32)
    cache.append(k, v, seq.cuda(), pos.cuda(), table.cuda())
    check_codes(cache, params, table, k.cpu(), v.cpu(), seq, pos, theta=None)
    # heads-first storage, rows that do not start on 16 bytes, 64-bit indexes, a wider table
    odd = torch.randn(3, 77, D + 1, generator=g).to(torch.bfloat16).cuda()[:, :, 1:].transpose(0, 1)
    big = torch.full((2, 6), -1, dtype=torch.int64)
    big[:, 1:4] = table
    cache.append(odd, v, seq.long().cuda(), pos.long().cuda(), big.cuda()[:1, 1:4])
    check_codes(cache, params, table, odd.cpu(), v.cpu(), seq, pos, theta=None)
    one = torch.randn(77, 1, D, generator=g).cuda().expand(77, 3, D)  # one key head for all, stride 0
    cache.append(one, one, seq.cuda(), pos.cuda(), table.cuda())
    check_codes(cache, params, table, one.cpu(), one.cpu(), seq, pos, theta=None)
    cache.check()


@pytest.mark.gpu
def test_append_extremes():
    cache, params = make(2, 1, 16, theta=None)
    x = torch.zeros(10, 1, D)
    x[1, 0, 5] = 3.0                      # one coordinate
    x[2] = 1e30                           # squares overflow
    x[3] = 1e-30                          # squares underflow: reads as zero
    x[4, 0, 7] = float("nan")
    x[5, 0, 0] = float("inf")
    x[6] = 3e38                           # squares overflow
    x[7] = -1.0
    x[8, 0, :2] = 1.0
    x[9] = 1e5                            # norm past fp16: capped
    at = torch.arange(10, dtype=torch.int32)
    zero = torch.zeros(10, dtype=torch.int32).cuda()
    cache.append(x.cuda(), x.cuda(), zero, at.cuda(), torch.tensor([[1]], dtype=torch.int32).cuda())
    for t in cache.read(zero, at.cuda(), torch.tensor([[1]], dtype=torch.int32).cuda(), dtype=torch.float32):
        t = t.cpu()
        assert (t[0] == 0).all() and (t[3] == 0).all()
        assert t[9].norm().item() == pytest.approx(65504.0, rel=0.15) and torch.isfinite(t[9]).all()
        for i in (2, 4, 5, 6):
            assert torch.isnan(t[i]).all()
        for i in (1, 7, 8):  # all of a rotated vector's weight on few levels: quantised coarsely, but the right way
            assert torch.nn.functional.cosine_similarity(t[i].flatten(), x[i].flatten(), 0) > 0.9


# ------------------------------------------------------------------------------------ read --
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,page_size,norm", [(1, 16, "float16"), (5, 64, "bfloat16"), (12, 128, "float16")])
def test_read(dtype, heads, page_size, norm):
    cache, params, table, (k, v, seq, pos, _) = filled([1, 133, 70], heads, page_size, norm, mask_every=5)
    pick = torch.randperm(len(seq), generator=torch.Generator().manual_seed(2))[:101]
    got = cache.read(seq[pick].cuda(), pos[pick].cuda(), table.cuda(), dtype=dtype)
    pg, off = table[seq[pick].long(), pos[pick].long() // page_size].long(), pos[pick].long() % page_size
    full = got if dtype == torch.float32 else cache.read(seq[pick].cuda(), pos[pick].cuda(), table.cuda(),
                                                        dtype=torch.float32)
    for which in range(2):
        want, _ = stands_for(cache, params[which], which)
        want = want[pg, off]
        # fp32: seven roundings of sums of 64 levels; bf16: those, rounded once
        tol = want.norm(dim=-1, keepdim=True) * 2.0 ** -21
        assert ((full[which].double().cpu() - want).abs() <= tol).all()
        assert torch.equal(got[which], full[which].to(dtype))
    # what it stands for is near what went in: 4 bits leave about 0.1 of the norm
    x = v[pick].double()
    err = (got[1].double().cpu() - x).norm(dim=-1) / x.norm(dim=-1)
    assert err.mean() < 0.11 and err.max() < 0.25


@pytest.mark.gpu
def test_cache_holds_what_the_hook_simulates():
    """The TurboQuant hook on the same rows and quantisers, its codebook made even as the cache's is (the Lloyd-Max
    iteration leaves the halves up to 6.1e-5 apart, which moves about one decision in a thousand)."""
    from cutechronos_b200 import turboquant as tq
    cache, params = make(4, 4, 64, theta=None)
    g = torch.Generator().manual_seed(9)
    rows = torch.randn(130, 3 * 4 * D, generator=g).cuda()
    seq, pos = torch.zeros(130, dtype=torch.int32).cuda(), torch.arange(130, dtype=torch.int32).cuda()
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32).cuda()
    cache.append(rows[:, 256:512].view(130, 4, D), rows[:, 512:].view(130, 4, D), seq, pos, table)
    got = cache.read(seq, pos, table, dtype=torch.float32)
    kp, vp = (tq.TurboQuantParams.build(D, 4, mode="mse", seed=s) for s in (3, 4))
    for p in (kp, vp):
        lv, bounds, _, _ = tables(p)
        p.tensors["codebook"] = torch.cat([-lv.flip(0), lv]).float().cuda()
        p.tensors["boundaries"] = torch.cat([-bounds.flip(0), torch.zeros(1), bounds]).float().cuda()
    tq.kv_quant(rows, 130, 4, kp, vp, q_col=0, k_col=256, v_col=512)
    for t, col in zip(got, (256, 512)):
        ref = rows[:, col:col + 256].view(130, 4, D)
        assert ((t - ref).norm(dim=-1) / ref.norm(dim=-1)).median() < 5e-4
        assert (t - ref).norm() / ref.norm() < 5e-3


# ------------------------------------------------------------------------------- attention --
def run_case(lens, new, heads, group, page_size=64, norm="float16", dtype=torch.bfloat16, causal=True, rotate=True,
             scale=0.125, mask_every=0, seed=0, uniform=False, **kw):
    cache, params, table, _ = filled(lens, heads, page_size, norm, dtype, seed, mask_every)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    g = torch.Generator().manual_seed(seed + 100)
    q = (torch.randn(cu[-1], heads * group, D, generator=g) * 1.5).to(dtype)
    args = dict(causal=causal, scale=scale, rotate_q=rotate, return_lse=True, **kw)
    if not uniform:
        args.update(cu_q=torch.tensor(cu, dtype=torch.int32).cuda(), max_q=max(new))
    out, lse = cache.attention(q.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), table.cuda(), **args)
    want, wlse, sway, weight = oracle_attention(cache, params, q, lens, table, cu, causal, scale, rotate)
    tol, ltol = allowed(want, sway, weight, dtype == torch.float32)
    err = (out.double().cpu() - want).norm(dim=-1)
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), (err / tol).max()
    empty = wlse == -math.inf
    got = lse.double().cpu()
    assert torch.equal(got == -math.inf, empty)
    assert ((got - wlse).abs()[~empty] <= ltol[~empty]).all()
    assert (out.cpu()[empty] == 0).all()
    # as a whole the rounding is random: far below what a single row may be off
    assert err.norm() / want.norm().clamp(min=1e-30) <= (2.0 ** -17 if dtype == torch.float32 else 2.0 ** -8) or want.norm() == 0
    cache.check()
    return out, lse


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 256])
def test_single_token_every_length(page_size, dtype):
    lens = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 129, 255, 256, 257, 600]
    run_case(lens, [1] * len(lens), 2, 1, page_size, dtype=dtype, uniform=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads,group", [(1, 1), (12, 1), (3, 4), (2, 7), (1, 8), (1, 12), (2, 17), (1, 40)])
def test_single_token_head_layouts(heads, group, dtype):
    run_case([133, 700], [1, 1], heads, group, dtype=dtype, norm="bfloat16")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new", [[2, 3, 2], [9, 1, 0], [33, 5, 17], [130, 64, 1], [300, 129, 257]])
def test_several_tokens(new, causal, dtype):
    run_case([513, 70, 300], new, 2, 3, 32, dtype=dtype, causal=causal, mask_every=7)


@pytest.mark.gpu
@pytest.mark.parametrize("rotate", [True, False])
@pytest.mark.parametrize("lens,new", [([4000], [1]), ([3333, 1], [2, 1]), ([2500, 4000], [150, 700])])
def test_long_axis_is_split_and_joined(lens, new, rotate):
    run_case(lens, new, 2, 2, rotate=rotate)
    run_case(lens, new, 2, 2, rotate=rotate, max_len=4096 * 4, mask_every=3)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 5, 40, 200])
def test_more_queries_than_keys(new):
    """Rows that stand before the sequence's first entry see nothing when causal."""
    run_case([new // 2, 0, 3], [new, new, new], 2, 2, uniform=True)
    run_case([new // 2, 0, 3], [new, new, new], 2, 2, uniform=True, causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 20, 140])
def test_all_tokens_masked(new):
    cache, params, table, (k, v, seq, pos, _) = filled([70, 200], 2)
    cache.append(k.cuda(), v.cuda(), seq.cuda(), pos.cuda(), table.cuda(), token_mask=(seq == 1).cuda())
    q = torch.randn(2 * new, 2, D, dtype=torch.bfloat16, device="cuda")
    out, lse = cache.attention(q, torch.tensor([70, 200], dtype=torch.int32).cuda(), table.cuda(), return_lse=True,
                               causal=False)
    assert (out[:new] == 0).all() and (lse[:new] == -math.inf).all()
    assert torch.isfinite(lse[new:]).all() and (out[new:] != 0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 9, 140])
def test_what_is_masked_or_not_finite_stays_out(new, dtype):
    """NaN and infinite keys and values at masked tokens change nothing; at visible ones they make the rows that see
    them NaN, and only those."""
    cache, params, table, (k, v, seq, pos, _) = filled([200], 2, dtype=dtype)
    q = torch.randn(new, 2, D, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    lens, tab = torch.tensor([200], dtype=torch.int32).cuda(), table.cuda()
    mask = (pos != 17) & (pos != 198)
    cache.append(k.cuda(), v.cuda(), seq.cuda(), pos.cuda(), tab, token_mask=mask.cuda())
    ref = cache.attention(q, lens, tab)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[17], bad_v[17], bad_k[198], bad_v[198] = float("nan"), float("inf"), float("inf"), float("nan")
    cache.append(bad_k.cuda(), bad_v.cuda(), seq.cuda(), pos.cuda(), tab, token_mask=mask.cuda())
    assert torch.equal(ref, cache.attention(q, lens, tab))
    cache.append(k.cuda(), bad_v.cuda(), seq.cuda(), pos.cuda(), tab, token_mask=(pos != 17).cuda())
    out = cache.attention(q, lens, tab)
    late = 200 - new + torch.arange(new) >= 198
    assert torch.isnan(out[late.cuda()]).all()
    assert torch.equal(out[~late.cuda()], cache.attention(q, lens, tab)[~late.cuda()])
    assert torch.isfinite(out[~late.cuda()]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 140])
@pytest.mark.parametrize("qs,vs", [(1e4, 1.0), (1e-12, 1e-7), (1.0, 1e4), (1e-3, 1e-4)])
def test_scale_of_queries_and_values(qs, vs, new, dtype):
    """Sizes that fp16 alone would lose are scaled by powers of two on the way: only what the norm's fp16 loses shows."""
    cache, params = make(4, 1, 64, norm="bfloat16", theta=None)
    g = torch.Generator().manual_seed(8)
    k, v = torch.randn(150, 1, D, generator=g), torch.randn(150, 1, D, generator=g) * vs
    v[:75] *= 1e-2
    seq, pos = torch.zeros(150, dtype=torch.int32), torch.arange(150, dtype=torch.int32)
    table = torch.tensor([[3, 1, 0]], dtype=torch.int32)
    cache.append(k.cuda(), v.cuda(), seq.cuda(), pos.cuda(), table.cuda())
    q = (torch.randn(new, 2, D, generator=g) * qs).to(dtype)
    scale = 0.2 / qs
    out = cache.attention(q.cuda(), torch.tensor([150], dtype=torch.int32).cuda(), table.cuda(), scale=scale)
    want, _, sway, weight = oracle_attention(cache, params, q, [150], table, [0, new], True, scale, False)
    tol, _ = allowed(want, sway, weight, dtype == torch.float32)
    assert ((out.double().cpu() - want).norm(dim=-1) <= tol).all()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Pages beyond 4 GiB of the pool; every byte offset is 64 bits wide."""
    heads, ps = 12, 256
    page_bytes = heads * ps // 16 * 1088
    pages = (1 << 32) // page_bytes + 40
    cache, params = make(pages, heads, ps, max_positions=2048)
    g = torch.Generator().manual_seed(1)
    lens = [600, 300]
    table = torch.tensor([[pages - 1, pages - 7, pages - 3], [pages - 2, pages - 20, -1]], dtype=torch.int32)
    seq = torch.cat([torch.zeros(600), torch.ones(300)]).int()
    pos = torch.cat([torch.arange(600), torch.arange(300)]).int()
    k, v = (torch.randn(900, heads, D, generator=g).to(torch.bfloat16) for _ in range(2))
    cache.append(k.cuda(), v.cuda(), seq.cuda(), pos.cuda(), table.cuda())
    small, _ = make(6, heads, ps, max_positions=2048)
    near = torch.tensor([[5, 1, 3], [4, 0, -1]], dtype=torch.int32)
    small.append(k.cuda(), v.cuda(), seq.cuda(), pos.cuda(), near.cuda())
    for a, b in zip(cache.read(seq.cuda(), pos.cuda(), table.cuda()), small.read(seq.cuda(), pos.cuda(), near.cuda())):
        assert torch.equal(a, b)
    n = torch.tensor(lens, dtype=torch.int32).cuda()
    for new in (1, 150):
        q = torch.randn(2 * new, heads, D, generator=g).to(torch.bfloat16).cuda()
        assert torch.equal(cache.attention(q, n, table.cuda(), scale=0.125), small.attention(q, n, near.cuda(), scale=0.125))
    cache.check()


@pytest.mark.gpu
def test_strided_queries_and_outputs():
    cache, params, table, _ = filled([150, 90], 3)
    lens = torch.tensor([150, 90], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(6)
    packed = torch.randn(20, 3 * 6 * D, generator=g).to(torch.bfloat16).cuda()
    q = packed[:, :6 * D].view(20, 6, D)
    ref = cache.attention(q.contiguous(), lens, table.cuda())
    assert torch.equal(ref, cache.attention(q, lens, table.cuda()))
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    room = torch.zeros(6, 20, 2 * D, dtype=torch.bfloat16, device="cuda")
    out = cache.attention(heads_first, lens, table.cuda(), out=room[:, :, D:].transpose(0, 1))
    assert torch.equal(ref, out) and (room[:, :, :D] == 0).all()
    odd = torch.empty(20, 6, D + 1, dtype=torch.bfloat16, device="cuda")[:, :, 1:]
    odd.copy_(q)
    assert torch.equal(ref, cache.attention(odd, lens, table.cuda()))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 150])
def test_calls_repeat_bit_for_bit_and_on_other_streams(new):
    cache, params, table, (k, v, seq, pos, _) = filled([2000, 900], 2)
    lens = torch.tensor([2000, 900], dtype=torch.int32).cuda()
    q = torch.randn(2 * new, 4, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    ref = cache.attention(q, lens, table.cuda(), scale=0.125)
    side = [torch.cuda.Stream() for _ in range(2)]
    tab = table.cuda()
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(side[i % 2]):
            got.append(cache.attention(q, lens, tab, scale=0.125))
    torch.cuda.synchronize()
    assert all(torch.equal(ref, t) for t in got)
    d = [t.cuda() for t in (k, v, seq, pos)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(*d, tab)
        out = cache.attention(q, lens, tab, scale=0.125)
    lens.copy_(torch.tensor([1900, 33], dtype=torch.int32))
    graph.replay()
    assert torch.equal(out, cache.attention(q, lens, tab, scale=0.125))


@pytest.mark.gpu
def test_refusals():
    cache, _ = make(8, 4, 32, max_positions=100)
    dev = dict(device="cuda", dtype=torch.int32)
    k = torch.zeros(5, 4, D, dtype=torch.bfloat16, device="cuda")
    seq, pos, table = torch.zeros(5, **dev), torch.arange(5, **dev), torch.arange(8, **dev).view(2, 4)
    lens = torch.tensor([5, 5], **dev)
    for err, call in (
            (RuntimeError, lambda: cache.append(k.cpu(), k, seq, pos, table)),
            (ValueError, lambda: cache.append(k[:, :3], k[:, :3], seq, pos, table)),
            (ValueError, lambda: cache.append(k, k[:4], seq, pos, table)),
            (ValueError, lambda: cache.append(k, k.float(), seq, pos, table)),
            (TypeError, lambda: cache.append(k.half(), k.half(), seq, pos, table)),
            (ValueError, lambda: cache.append(k[..., :32], k[..., :32], seq, pos, table)),
            (ValueError, lambda: cache.append(k, k, seq[:4], pos, table)),
            (TypeError, lambda: cache.append(k, k, seq.float(), pos, table)),
            (ValueError, lambda: cache.append(k, k, seq, pos, table[0])),
            (ValueError, lambda: cache.append(k, k, seq, pos, table, token_mask=torch.ones(4, device="cuda"))),
            (TypeError, lambda: cache.read(seq, pos, table, dtype=torch.float16)),
            (ValueError, lambda: cache.attention(k, lens, table[:1])),
            (ValueError, lambda: cache.attention(k, lens, table)),               # 5 rows for 2 sequences
            (ValueError, lambda: cache.attention(k[:4, :3], lens, table)),       # 3 heads over 4
            (ValueError, lambda: cache.attention(k, lens, table, cu_q=lens)),
            (ValueError, lambda: cache.attention(k[:4], lens, table, out=k[:4].float())),
            (ValueError, lambda: cache.attention(k[:4], lens, table, out=k[:1].expand(4, 4, D))),
            (nat.NativeError, lambda: cache.attention(k[:4], lens, table, scale=float("nan"))),
            (ValueError, lambda: make(4, 4, theta=None)[0].attention(k[:4], lens, table, rotate_q=True))):
        with pytest.raises(err):
            call()
    # empty calls are fine
    cache.append(k[:0], k[:0], seq[:0], pos[:0], table)
    assert cache.read(seq[:0], pos[:0], table)[0].shape == (0, 4, D)
    assert cache.attention(k[:0], lens, table).shape == (0, 4, D)
    cache.check()


@pytest.mark.gpu
def test_out_of_range_is_skipped_and_reported():
    cache, _ = make(4, 2, 16, max_positions=40)
    dev = dict(device="cuda", dtype=torch.int32)
    table = torch.tensor([[0, 1, 2], [3, 77, -5]], **dev)
    before = cache.pages.clone()
    k = torch.randn(1, 2, D, device="cuda")
    for seq, pos, bad in ((-1, 3, False), (0, -1, False), (2, 0, True), (0, 48, True), (0, 45, True), (1, 16, True),
                          (1, 32, True)):
        s, p = torch.tensor([seq], **dev), torch.tensor([pos], **dev)
        cache.append(k, k, s, p, table)
        if bad:
            with pytest.raises(nat.NativeError, match="out of range"):
                cache.check()
        cache.check()
        if pos != 45:
            assert (cache.read(s, p, table)[0] == 0).all()
            if bad:
                with pytest.raises(nat.NativeError):
                    cache.check()
        assert torch.equal(before, cache.pages)
    q = torch.zeros(2, 2, D, device="cuda")
    for lens in ([49, 1], [-1, 1], [16, 17]):
        cache.attention(q, torch.tensor(lens, **dev), table)
        with pytest.raises(nat.NativeError, match="out of range"):
            cache.check()
    cache.attention(q, torch.tensor([48, 16], **dev), table)
    cache.check()


@pytest.mark.gpu
def test_model_cache_and_streaming_example():
    import importlib.util
    from pathlib import Path

    from conftest import small_config
    spec = importlib.util.spec_from_file_location(
        "streaming_attention", Path(__file__).resolve().parents[1] / "examples" / "streaming_attention.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.main(series=3, context=500, steps=9, page_size=16, layer=1, config=small_config())
    assert got["output"].shape == got["reference"].shape == (3, 32, 2, 64)
    # 4 bits leave 0.1 of a vector's norm; averages over keys less, the first tokens' rows most of it
    assert got["error"] < 0.12 and got["ratio"] > 3.7
    assert torch.isfinite(got["update"].float()).all()


def test_model_cache_refuses_bad_layers():
    from conftest import small_config
    from cutechronos_b200.model import CuteChronos2Model
    with pytest.raises(ValueError, match="layer"):
        CuteChronos2Model(small_config()).kv4_cache(4, layer=2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        CuteChronos2Model(small_config()).kv4_cache(4)


# ------------------------------------------------------- blocks, tiles and roundings of their own --
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [1, 2, 3, 5, 7, 12])
def test_append_and_read_every_block_shape(heads, dtype):
    """Calls whose tokens and heads fill no block of 16 tokens x 4 heads, or run over one, in a shuffled order, against
    one call with all tokens."""
    cache, params, table, (k, v, seq, pos, _) = filled([67], heads, 16, dtype=dtype)
    check_codes(cache, params, table, k, v, seq, pos)
    there = cache.read(seq.cuda(), pos.cuda(), table.cuda(), dtype=dtype)
    for n in (1, 2, 15, 16, 17, 31, 33, 50):
        o = torch.randperm(67, generator=torch.Generator().manual_seed(n))[:n]
        part, _ = make(cache.num_pages, heads, 16)
        part.pages.fill_(0xFF)
        part.append(k[o].cuda(), v[o].cuda(), seq[o].cuda(), pos[o].cuda(), table.cuda())
        rest = torch.ones(67, dtype=torch.bool).index_fill(0, o, False)
        part.append(k[rest].cuda(), v[rest].cuda(), seq[rest].cuda(), pos[rest].cuda(), table.cuda())
        assert torch.equal(part.pages, cache.pages)
        for a, b in zip(there, part.read(seq[o].cuda(), pos[o].cuda(), table.cuda(), dtype=dtype)):
            assert torch.equal(a[o.cuda()], b)
    cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
def test_tiles_that_leave_lanes_unused(causal):
    """Rows that fill one, two, three or all quarters of a tile's lanes, in many items, so that blocks go from one to
    the next with tiles that start elsewhere."""
    new = [11, 22, 32, 33, 43, 54, 64, 75, 86, 96] * 4
    lens = [n + 7 * (i % 11) for i, n in enumerate(new)]
    run_case(lens, new, 5, 3, 16, causal=causal, mask_every=9)


@pytest.mark.gpu
@pytest.mark.parametrize("group,new", [(1, 1), (4, 1), (4, 2), (4, 4)])
def test_rounding_of_a_long_context(group, new):
    """Up to 16 rows, what a bf16 call adds to the rounding of its output is small.  Scores of deviation 4: the levels'
    rounding, 0.95e-4 of each weighted by its share of a vector, moves weights by about 4e-4 (K) and V^ by 1e-4, P's by
    1.4e-4; next to the output's own 1.65e-3 that makes 1.03 of it.  One fp16 part of Q would add 1e-3 and make 1.2."""
    cache, params, table, _ = filled([20000], 2, 64, theta=None, seed=21)
    g = torch.Generator().manual_seed(22)
    k = torch.randn(20000, 2, D, generator=g)
    v = torch.randn(20000, 2, D, generator=g)
    ids = torch.zeros(20000, dtype=torch.int32), torch.arange(20000, dtype=torch.int32)
    cache.append(k.cuda(), v.cuda(), *(t.cuda() for t in ids), table.cuda())
    q = torch.randn(new, 2 * group, D, generator=g).to(torch.bfloat16)
    lens = torch.tensor([20000], dtype=torch.int32).cuda()
    got = cache.attention(q.cuda(), lens, table.cuda(), scale=0.5, causal=True).double().cpu()
    want, *_ = oracle_attention(cache, params, q, [20000], table, [0, new], True, 0.5, False)
    own = (want.to(torch.bfloat16).double() - want).norm()
    assert (got - want).norm() <= 1.12 * own


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("norm", ["float16", "bfloat16"])
def test_17_to_32_rows_of_long_sequences(norm, causal):
    """Beside the same rows of short sequences, which another kernel takes."""
    new = [13, 16, 9, 0, 1, 15]
    run_case([1500, 1100, 64, 5, 1, 1030], new, 2, 2, 32, norm, causal=causal, mask_every=7)
    run_case([500, 1000, 64, 5, 1, 530], new, 2, 2, 32, norm, causal=causal, mask_every=7)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [3, 60])
def test_row_bounds_that_fall_or_overlap(rows, dtype):
    """cu_q is device data that a call cannot check before it launches: bounds that fall, run past the rows or name the
    same rows for many sequences leave unspecified rows, nothing else; a call after them is right."""
    n = 12
    cache, params, table, _ = filled([700] * n, 2, dtype=dtype)
    lens = torch.full((n,), 700, dtype=torch.int32).cuda()
    total = n * rows
    q = torch.randn(total, 4, D, generator=torch.Generator().manual_seed(9)).to(dtype).cuda()
    pages = cache.pages.clone()
    good = torch.arange(0, total + 1, rows, dtype=torch.int32)
    args = dict(max_q=total, scale=0.125, rotate_q=True)
    want = cache.attention(q, lens, table.cuda(), cu_q=good.cuda(), **args)
    falling = good.clone()
    falling[0], falling[3], falling[7] = total // 2, 0, total + 50
    again = torch.tensor([0, total] * (n // 2) + [0], dtype=torch.int32)
    backwards = good.flip(0).contiguous()
    for cu in (falling, again, backwards, torch.full_like(good, -7), torch.full_like(good, 2**31 - 1)):
        out = torch.empty(total + 64, 4, D, dtype=dtype, device="cuda").fill_(7)
        cache.attention(q, lens, table.cuda(), cu_q=cu.cuda(), out=out[32:-32], **args)
        assert (out[:32] == 7).all() and (out[-32:] == 7).all()
        with pytest.raises(nat.NativeError, match="out of range"):
            cache.check()
        assert torch.equal(cache.pages, pages)
        assert torch.equal(cache.attention(q, lens, table.cuda(), cu_q=good.cuda(), **args), want)
        cache.check()
