"""Edges of the paged 4-bit K/V cache: what lies beside a call's operands, values at the ends of their range, and the
errors that calls leave for :meth:`PagedKV4Cache.check`."""

from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

from cutechronos_b200 import _native as nat
from test_kvcache import D, allowed, filled, make, oracle_attention, tables, unpack, walsh

I32 = dict(device="cuda", dtype=torch.int32)


# ------------------------------------------------------------------ a block table within a wider one --
def test_calls_are_bounded_by_a_tables_columns():
    """What append and read hand to the library for a table of three columns within one of six: rows 6 apart, 3 long."""
    from cutechronos_b200.kvcache import PagedKV4Cache

    class Recorded(PagedKV4Cache):
        def __init__(self):
            self._at, self.device, self.num_heads, self.page_size = -1, torch.device("cpu"), 2, 16
            self._lib = nat.load()

        def _call(self, fn, what, *args):
            self.last = args

    cache = Recorded()
    big = torch.arange(18, dtype=torch.int32).view(3, 6)
    k = torch.zeros(5, 2, D)
    seq, pos = torch.zeros(5, dtype=torch.int32), torch.arange(5, dtype=torch.int32)
    for table, ld in ((big[:, 3:6], 6), (big[:1, 3:6], 3), (big[:, 3:6].clone(), 3), (big[:1, 3:6].expand(3, 3), 3)):
        cache.append(k, k, seq, pos, table)
        assert cache.last[-3:] == (ld, 3, table.shape[0])
        cache.read(seq, pos, table)
        assert cache.last[-3:] == (ld, 3, table.shape[0])


def test_table_columns_are_checked():
    lib = nat.load()
    c = nat.KV4Cache(pages=1 << 20, num_pages=4, page_size=64, heads=2)
    r = C.byref(c)
    for ld, cols in ((4, 5), (4, 0), (0, 0), (4, -1)):
        assert lib.cc2_kv4_append_cols(r, 1, 1 << 20, 128, 64, 1 << 20, 128, 64, 1, 64, 64, None, 64, ld, cols, 1, None) == -1
        assert b"block table" in lib.cc2_last_error()
        assert lib.cc2_kv4_read_cols(r, 1, 1 << 20, 1 << 20, 1, 64, 64, 64, ld, cols, 1, None) == -1
        assert b"block table" in lib.cc2_last_error()


@pytest.mark.gpu
def test_positions_past_a_sliced_tables_columns():
    """They are skipped and reported: neither the next row's pages nor what lies past the table is touched."""
    cache, _ = make(18, 2, 16, max_positions=400)
    big = torch.arange(18, **I32).view(3, 6)
    table = big[:, 3:6]
    g = torch.Generator().manual_seed(1)
    k = torch.randn(1, 2, D, generator=g).cuda()
    before = cache.pages.clone()
    for s in range(3):
        for p in (48, 63, 95, 399):
            seq, pos = torch.tensor([s], **I32), torch.tensor([p], **I32)
            cache.append(k, k, seq, pos, table)
            with pytest.raises(nat.NativeError, match="out of range"):
                cache.check()
            assert torch.equal(before, cache.pages)
            assert all((t == 0).all() for t in cache.read(seq, pos, table))
            with pytest.raises(nat.NativeError, match="out of range"):
                cache.check()
    # what lies in the columns goes where a table of its own would put it
    own, _ = make(18, 2, 16, max_positions=400)
    seq = torch.arange(3, **I32).repeat_interleave(48)
    pos = torch.arange(48, **I32).repeat(3)
    k, v = (torch.randn(144, 2, D, generator=g).cuda() for _ in range(2))
    cache.append(k, v, seq, pos, table)
    own.append(k, v, seq, pos, table.contiguous())
    assert torch.equal(cache.pages, own.pages) and not torch.equal(cache.pages, before)
    for a, b in zip(cache.read(seq, pos, table), own.read(seq, pos, table.contiguous())):
        assert torch.equal(a, b)
    cache.check()


def test_rotation_table_must_be_aligned():
    """The kernels read it 16 bytes at a time."""
    lib = nat.load()
    n = C.c_size_t()
    c = nat.KV4Cache(pages=1 << 20, num_pages=4, page_size=64, heads=2, rope_cs=(1 << 20) + 8, rope_len=16)
    assert lib.cc2_kv4_attention_workspace_bytes(C.byref(c), 1, 2, 1, 1, 1, 64, C.byref(n)) == -1
    assert b"rope_cs must be 16-byte aligned" in lib.cc2_last_error()
    c.rope_cs = 1 << 20
    assert lib.cc2_kv4_attention_workspace_bytes(C.byref(c), 1, 2, 1, 1, 1, 64, C.byref(n)) == 0


# -------------------------------------------------------------------- scores and values at their ends --
def against_oracle(cache, params, table, q, lens, new, scale, sway=None, causal=True):
    """Output and log-sum-exp of a call next to the 64-bit ones, within ``allowed``; as a whole the rounding is random."""
    f32 = q.dtype == torch.float32
    out, lse = cache.attention(q.cuda(), torch.tensor(lens, **I32), table.cuda(), scale=scale, causal=causal, return_lse=True)
    want, wlse, most, weight = oracle_attention(cache, params, q, lens, table, [i * new for i in range(len(lens) + 1)],
                                                causal, scale, False)
    tol, ltol = allowed(want, most if sway is None else sway, weight, f32)
    assert torch.isfinite(out).all()
    err = (out.double().cpu() - want).norm(dim=-1)
    assert (err <= tol).all(), (err / tol).max()
    assert err.norm() <= want.norm() * (2.0 ** -17 if f32 else 2.0 ** -8)
    empty, lse = wlse == -math.inf, lse.double().cpu()
    assert torch.equal(lse == -math.inf, empty) and (out.cpu()[empty] == 0).all()
    assert ((lse - wlse).abs()[~empty] <= ltol[~empty]).all()
    cache.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 20, 40, 200])
@pytest.mark.parametrize("zero", ["queries", "scale", "all"])
@pytest.mark.parametrize("what", ["masked", "keys", "masked and keys", "all masked"])
def test_scores_of_zero_beside_blocks_of_masked_or_zero_keys(what, zero, new, dtype):
    """Rows of zeros, a scale of zero, or both, over blocks of 128 keys that are all masked, of zero norm, or both: the
    mean of the values that a row sees, and nothing where it sees none."""
    n = 400
    cache, params = make(8, 2, 64, theta=None)
    g = torch.Generator().manual_seed(31)
    k, v = (torch.randn(n, 2, D, generator=g) for _ in range(2))
    q = torch.randn(new, 4, D, generator=g)
    at = torch.arange(n, dtype=torch.int32)
    mask = torch.ones(n, dtype=torch.bool)
    if "masked" in what:
        mask[:256] = False  # two whole blocks, and their rows' only keys
    if what == "all masked":
        mask[:] = False
    if "keys" in what:
        k[200:] = 0.0       # the rest of a block, a whole one and a last one of 16 keys
    if zero != "scale":
        q[::2] = 0.0
    if zero == "all":
        q[:] = 0.0
    table = torch.tensor([[5, 1, 0, 7, 2, 6, 3]], dtype=torch.int32)
    cache.append(k.to(dtype).cuda(), v.to(dtype).cuda(), torch.zeros(n, **I32), at.cuda(), table.cuda(),
                 token_mask=mask.cuda())
    against_oracle(cache, params, table, q.to(dtype), [n], new, 0.0 if zero == "scale" else 0.125)


def spread_case(spread, where, new, dtype):
    """300 keys of norm about 1, of values of norm 2^(15 - spread), but for one of norm 2^15 that has no weight (a key far
    against the queries' common direction) or that only the last row could see."""
    n, at = 300, {"first block": 3, "second block": 200, "last": 299}[where]
    cache, params = make(6, 1, 64, theta=None)
    g = torch.Generator().manual_seed(41)
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)  # noqa: E731
    u = unit(torch.randn(D, generator=g))
    k, v = unit(torch.randn(n, 1, D, generator=g)), unit(torch.randn(n, 1, D, generator=g)) * 2.0 ** (15 - spread)
    k[at], v[at] = -60 * u, v[at] * 2.0 ** spread
    q = (unit(torch.randn(new, 2, D, generator=g)) + 2 * u).to(dtype)
    table = torch.tensor([[4, 1, 0, 5, 2]], dtype=torch.int32)
    cache.append(k.to(dtype).cuda(), v.to(dtype).cuda(), torch.zeros(n, **I32), torch.arange(n, **I32), table.cuda())
    # the one key's weight is under 2^-60: its score may be off by what it likes
    sway = q.double().norm(dim=-1) * 1.2
    against_oracle(cache, params, table, q, [n], new, 1.0, sway)


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["first block", "second block", "last"])
@pytest.mark.parametrize("new", [1, 7, 12, 20, 140])
@pytest.mark.parametrize("spread", [0, 10, 13, 16, 18, 20])
def test_one_value_far_larger_than_those_that_count(spread, new, where):
    spread_case(spread, where, new, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["first block", "second block", "last"])
@pytest.mark.parametrize("new", [1, 3, 7, 140])
@pytest.mark.parametrize("spread", [0, 10, 13, 16, 18, 20])
def test_one_value_far_larger_than_those_that_count_fp32(spread, new, where):
    spread_case(spread, where, new, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 9, 25, 140])
@pytest.mark.parametrize("bad", ["value", "key", "both"])
def test_not_finite_keys_and_values_reach_the_rows_that_see_them(bad, new, dtype):
    """A visible value that is not finite makes the rows that see it NaN and leaves their log-sum-exp, which has no value
    in it; a key makes both NaN.  Rows that do not see it stay what the clean cache gives, to within both roundings."""
    n = 200
    cache, params, table, (k, v, seq, pos, _) = filled([n], 2, dtype=dtype, theta=None)
    q = torch.randn(new, 2, D, generator=torch.Generator().manual_seed(4)).to(dtype)
    want, wlse, sway, weight = oracle_attention(cache, params, q, [n], table, [0, new], True, 0.125, False)
    tol, ltol = allowed(want, sway, weight, dtype == torch.float32)
    if bad != "key":
        v[198, 0, 3], v[198, 1, 60] = float("nan"), float("-inf")
    if bad != "value":
        k[198, 0, 3], k[198, 1, 60] = float("inf"), float("nan")
    cache.append(k.cuda(), v.cuda(), seq.cuda(), pos.cuda(), table.cuda())
    out, lse = (t.double().cpu() for t in cache.attention(q.cuda(), torch.tensor([n], **I32), table.cuda(), scale=0.125,
                                                          return_lse=True))
    late = n - new + torch.arange(new) >= 198
    assert torch.isnan(out[late]).all()
    assert ((out - want).norm(dim=-1) <= tol)[~late].all()
    near = (lse - wlse).abs() <= ltol
    if bad == "value":
        assert near.all()
    else:
        assert torch.isnan(lse[late]).all() and near[~late].all()


# ------------------------------------------------------------------------ whose error a status bit is --
def out_of_range(cache):
    """An append to a place that the cache does not have."""
    k = torch.zeros(1, cache.num_heads, D, device="cuda")
    cache.append(k, k, torch.zeros(1, **I32), torch.full((1,), 10**6, **I32), torch.zeros(1, 1, **I32))


@pytest.mark.gpu
def test_a_cache_error_is_not_the_forwards():
    """A checked forward succeeds beside a cache call that was out of range, and leaves the report of it to the cache."""
    from conftest import small_config
    from cutechronos_b200.model import CuteChronos2Model
    from cutechronos_b200.workloads import seeded_init_
    model = seeded_init_(CuteChronos2Model(small_config()), seed=1).to("cuda").eval().set_device_checks(True)
    x = torch.randn(2, 300, generator=torch.Generator().manual_seed(2)).cuda()
    want = model(x, num_output_patches=2).clone()
    cache, _ = make(2, 2, 16)
    cache.check()
    out_of_range(cache)
    assert torch.equal(want, model(x, num_output_patches=2))
    with pytest.raises(nat.NativeError, match="out of range"):
        cache.check()
    cache.check()


@pytest.mark.gpu
def test_a_cache_error_is_not_the_bridges(tmp_path):
    from conftest import small_config, write_checkpoint
    from cutechronos_b200.foreign import NativeBridge
    from cutechronos_b200.model import CuteChronos2Model
    from cutechronos_b200.workloads import seeded_init_
    write_checkpoint(seeded_init_(CuteChronos2Model(small_config()), seed=5), tmp_path)
    bridge = NativeBridge(nat.load())
    x = torch.randn(300, generator=torch.Generator().manual_seed(2)).tolist()
    h = bridge.init_pipeline(str(tmp_path))
    try:
        want, _ = bridge.predict_median(h, x, 16)
        cache, _ = make(2, 2, 16)
        out_of_range(cache)
        got, _ = bridge.predict_median(h, x, 16)
    finally:
        bridge.destroy_pipeline(h)
    assert want == got
    with pytest.raises(nat.NativeError, match="out of range"):
        cache.check()
    cache.check()


@pytest.mark.gpu
def test_a_forwards_timeout_is_not_the_caches():
    """The hook that withholds a load, as in the failure path's own test: the GEMM gives up after its bounded wait."""
    from cutechronos_b200 import kernels
    lib = nat.load()
    x, w = torch.randn(64, 768, device="cuda").to(torch.bfloat16), torch.randn(512, 768, device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    assert lib.cc2_device_status(1) == 0
    cache, _ = make(2, 2, 16)
    nat.check(lib.cc2_test_starve_gemm(1), "cc2_test_starve_gemm")
    try:
        kernels.linear(x, w)
        torch.cuda.synchronize()
        cache.check()
        assert lib.cc2_device_status(1) == 1
    finally:
        nat.check(lib.cc2_test_starve_gemm(0), "cc2_test_starve_gemm")
        lib.cc2_device_status(1)


@pytest.mark.gpu
def test_each_side_reads_and_resets_its_own_bits():
    lib = nat.load()
    cache, _ = make(2, 2, 16)
    assert lib.cc2_device_status(1) == 0
    out_of_range(cache)
    assert lib.cc2_device_status_of(nat.DEV_FORWARD, 1) == 0
    assert lib.cc2_device_status_of(nat.DEV_CACHE, 0) == nat.DEV_CACHE_RANGE
    assert lib.cc2_device_status(0) == nat.DEV_CACHE_RANGE
    assert lib.cc2_device_status(1) == nat.DEV_CACHE_RANGE
    assert lib.cc2_device_status(0) == 0
    cache.check()


# ------------------------------------------------------------------------------------ 64-bit indexes --
@pytest.mark.gpu
def test_64_bit_indexes_do_not_wrap():
    """An index that 32 bits would turn into a valid one is out of range, or, where it is negative, skips."""
    cache, _ = make(4, 2, 16, max_positions=64)
    I64 = dict(device="cuda", dtype=torch.int64)
    table = torch.tensor([[0, 1, 2, 3]], **I64)
    zero, at = torch.zeros(1, **I64), torch.tensor([5], **I64)
    k = torch.randn(1, 2, D, device="cuda")
    before = cache.pages.clone()

    def reported(yes=True):
        if yes:
            with pytest.raises(nat.NativeError, match="out of range"):
                cache.check()
        cache.check()

    for seq, pos, tab, bad in ((zero, at + 2**32, table, True), (zero + 2**32, at, table, True), (zero, at, table + 2**32, True),
                               (zero, at - 2**63, table, False), (zero - 2**40, at, table, False), (zero, at, table - 2**32, True)):
        cache.append(k, k, seq, pos, tab)
        reported(bad)
        assert torch.equal(before, cache.pages)
        assert all((t == 0).all() for t in cache.read(seq, pos, tab))
        reported(bad)
    cache.append(k, k, zero, at, table)
    assert not torch.equal(before, cache.pages)
    q = torch.randn(1, 2, D, device="cuda")
    want = cache.attention(q, torch.tensor([6], **I64), table)
    reported(False)
    cache.attention(q, torch.tensor([6 + 2**32], **I64), table)
    reported()
    cache.attention(q, torch.tensor([6], **I64), table, cu_q=torch.tensor([2**32, 2**32 + 1], **I64))
    reported()
    assert torch.equal(want, cache.attention(q, torch.tensor([6], **I32), table.int()))


@pytest.mark.gpu
def test_64_bit_indexes_of_any_strides():
    cache, _, table, (_, _, seq, pos, _) = filled([300, 90, 700], 2)
    tab = table.cuda()
    ref = cache.read(seq.cuda(), pos.cuda(), tab)
    wide = torch.full((3, 2 * table.shape[1] + 3), 2**40, dtype=torch.int64, device="cuda")
    wide[:, 1:-2:2] = tab
    pair = torch.stack([seq, pos], 1).long().cuda()
    for t in (tab.long(), wide[:, 1:-2:2], tab.long().t().contiguous().t()):
        for a, b in zip(ref, cache.read(pair[:, 0], pair[:, 1], t)):
            assert torch.equal(a, b)
    one = torch.zeros(1, dtype=torch.int64, device="cuda").expand(300)
    for a, b in zip(ref, cache.read(one, torch.arange(300, device="cuda"), tab[:1].long().expand(2, -1))):
        assert torch.equal(a[:300], b)
    assert cache.read(one[:0], one[:0], tab.long())[0].shape == (0, 2, D)
    cache.check()


# ----------------------------------------------------------------------------------------- tiny vectors --
@pytest.mark.gpu
@pytest.mark.parametrize("size", [3e-23, 4.4e-23, 6e-23, 1e-22, 1e-20, 1e-15])
def test_codes_of_vectors_whose_squares_underflow(size):
    """All of a vector's weight on one rotated coordinate: |y| = 8n passes every bound however the squares of fp32 round."""
    cache, params = make(1, 1, 16, norm="bfloat16", theta=None)
    _, _, signs, perm = tables(params[1])
    x = torch.zeros(4, 1, D)
    row = (walsh()[[0, 5, 38, 63]] * signs).float() * size
    x[:, 0, perm] = row
    x[2:] *= -1
    cache.append(x.cuda(), x.cuda(), torch.zeros(4, **I32), torch.arange(4, **I32), torch.zeros(1, 1, **I32))
    mag, sign, norm, _ = unpack(cache, 1)
    for i, j in enumerate((0, 5, 38, 63)):
        assert mag[0, i, 0, j] == 7 and sign[0, i, 0, j] == (1 if i < 2 else -1)
    assert (norm[0, :4, 0] > 0).all()


# -------------------------------------------------------------------------------- calls of two threads --
@pytest.mark.gpu
def test_a_call_keeps_the_plan_it_found():
    """Between a call's look at the cache's plan and its use, another thread's call may have left its own."""
    from cutechronos_b200.kvcache import PagedKV4Cache

    class Raced(PagedKV4Cache):
        @property
        def _plan(self):
            found, self.plan = self.plan, ((), 0)  # the other call's, which takes no workspace
            return found

        @_plan.setter
        def _plan(self, plan):
            self.plan = self.known = plan

    cache = Raced(64, 2, rope_theta=None)
    table = torch.arange(64, **I32).view(1, 64)
    k = torch.randn(3000, 2, D, device="cuda")
    cache.append(k, k, torch.zeros(3000, **I32), torch.arange(3000, **I32), table)
    q, lens = torch.randn(1, 2, D, device="cuda"), torch.tensor([3000], **I32)
    want = cache.attention(q, lens, table)
    assert cache.known[1] > 0
    cache.plan = cache.known
    assert torch.equal(want, cache.attention(q, lens, table))
    cache.check()


# ------------------------------------------------------------------------- rows that no sequence has --
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 5, 24, 150])
def test_rows_of_no_sequence(new, dtype):
    """Rows before cu_q's first entry and from its last on (a batch padded to a fixed size): 0 and -inf in a new output,
    left alone in one that the caller gives."""
    cache, _, table, _ = filled([300, 90, 700], 2, dtype=dtype)
    lens, tab = torch.tensor([300, 90, 700], **I32), table.cuda()
    total = 3 * new + 37
    q = torch.randn(total, 6, D, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    want, wlse = cache.attention(q[7:7 + 3 * new], lens, tab, scale=0.125, return_lse=True)
    cu = torch.tensor([7, 7 + new, 7 + 2 * new, 7 + 3 * new], **I32)
    args = dict(cu_q=cu, max_q=new, scale=0.125, return_lse=True)
    for fill in (7.0, float("nan")):
        stale = [torch.full_like(q, fill), torch.full((total, 6), fill, device="cuda")]
        del stale  # what a new output may be cut from
        out, lse = cache.attention(q, lens, tab, **args)
        assert torch.equal(out[7:7 + 3 * new], want) and torch.equal(lse[7:7 + 3 * new], wlse)
        for part in (slice(0, 7), slice(7 + 3 * new, None)):
            assert (out[part] == 0).all() and (lse[part] == -math.inf).all()
        room = torch.full_like(q, fill)
        got, lse = cache.attention(q, lens, tab, out=room, **args)
        assert torch.equal(got[7:7 + 3 * new], out[7:7 + 3 * new])
        for part in (slice(0, 7), slice(7 + 3 * new, None)):
            assert torch.equal(got[part].isnan(), room[part].isnan()) and (math.isnan(fill) or (got[part] == fill).all())
            assert (lse[part] == -math.inf).all()
    none, lse = cache.attention(q, lens, tab, cu_q=torch.full((4,), 9, **I32), max_q=0, return_lse=True)
    assert (none == 0).all() and (lse == -math.inf).all()
    cache.check()


@pytest.mark.gpu
def test_storage_is_written_not_replaced():
    """Calls go to the memory that the cache was made with: another tensor in its place would be passed over in silence."""
    cache, params = make(2, 2, 16)
    for name in ("pages", "rope"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name).clone())
    other, _ = make(2, 2, 16)
    k = torch.randn(16, 2, D, device="cuda")
    at = torch.zeros(16, **I32), torch.arange(16, **I32), torch.ones(1, 1, **I32)
    other.append(k, k, *at)
    cache.pages.copy_(other.pages)
    for a, b in zip(cache.read(*at), other.read(*at)):
        assert torch.equal(a, b) and (a != 0).any()
