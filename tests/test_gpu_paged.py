"""The paged plan, the paged QKV epilogue and the paged decode attention on the
GPU against their definitions (whole numbers exactly; values in 64 bits, with
the bounds that tests/_paged.py derives)."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

from _paged import LENGTH, NO_PAGE, PAGE_OOB, attention_ref, plan_ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from chatterbox_amdvulkan_b200 import ops as _ops
    return _ops


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------- plan --

def check_plan(p, ref, n_free_in=None):
    names = ("slots", "positions", "row_reqs", "row_lens", "row_start", "block_table", "n_blocks")
    for name, want in zip(names, ref):
        assert getattr(p, name).cpu().tolist() == want, name
    assert p.n_free.item() == ref[8]
    assert p.free_list.cpu().tolist() == ref[7]  # the popped entries behind the stack included
    assert p.err.item() == ref[9]


def pool(B, mb, P):
    return dict(table=[[-1] * mb for _ in range(B)], n_blocks=[0] * B, free=list(range(P)), n_free=P)


@pytest.mark.parametrize("B,page,ctx,spare", [(1, 16, 40, 0), (7, 1, 30, 5), (33, 5, 64, 10),
                                              (300, 16, 200, 100), (2100, 8, 50, 0)])
@pytest.mark.parametrize("mode", ["in_place", "new", "out"])
def test_plan_over_many_steps(ops, B, page, ctx, spare, mode):
    """A server's life: requests start, grow by 0..5 tokens, are cut back and end, over 8 steps."""
    r = random.Random(B * 7 + page)
    mb = -(-ctx // page)
    P = B * mb + spare
    st = pool(B, mb, P)
    r.shuffle(st["free"])
    dev = dict(block_table=ints(st["table"]), n_blocks=ints(st["n_blocks"]), free_list=ints(st["free"]),
               n_free=ints([P]))
    lens, out = [0] * B, None
    for _ in range(8):
        new = [0] * B
        for b in range(B):
            what = r.random()
            if what < 0.15:
                lens[b] = 0
            elif what < 0.3:
                lens[b] = new[b] = r.randint(1, ctx)
            elif what < 0.4:
                lens[b] = r.randint(0, lens[b])
            else:
                new[b] = min(r.randint(0, 5), ctx - lens[b])
                lens[b] += new[b]
        rows = sum(new) + r.choice((0, 0, 3))
        if mode == "out":
            rows = B * ctx // 2
        p = ops.paged_plan(ints(lens), **dev, page_size=page, n_new=ints(new), max_rows=rows,
                           in_place=mode == "in_place", out=out)
        ref = plan_ref(lens, new, st["table"], st["n_blocks"], st["free"], st["n_free"], page, rows)
        check_plan(p, ref)
        assert ref[9] in (0, LENGTH)
        assert (p.block_table.data_ptr() == dev["block_table"].data_ptr()) == (mode == "in_place")
        st = dict(table=ref[5], n_blocks=ref[6], free=ref[7], n_free=ref[8])
        if mode == "out":
            out = [torch.full_like(t, 99) for t in p[:9]]  # a second set of buffers, then the first again
        dev = dict(block_table=p.block_table, n_blocks=p.n_blocks, free_list=p.free_list, n_free=p.n_free)


def test_plan_decode_default_is_one_new_token(ops):
    lens = [3, 0, 17, 16]
    st = pool(4, 2, 9)
    p = ops.paged_plan(ints(lens), ints(st["table"]), ints(st["n_blocks"]), ints(st["free"]), ints([9]), 16)
    check_plan(p, plan_ref(lens, None, st["table"], st["n_blocks"], st["free"], 9, 16, 4))
    assert p.row_lens.tolist() == [3, 17, 16, 0]


@pytest.mark.parametrize("kw", [
    dict(lens=[20, 20, 20], new=[20, 20, 20], n_free=4),               # the pool runs dry
    dict(lens=[20, 1, 20], new=[1, 1, 1], n_free=0),                   # nothing at all
    dict(lens=[-3, 5, 2_000_000_000], new=[0, 5, 3]),                  # lengths outside
    dict(lens=[5, 6, 7], new=[-1, 9, 2]),                              # counts outside
    dict(lens=[5, 6, 7], new=[5, 6, 7], rows=8),                       # rows dropped
    dict(lens=[5, 6, 7], new=[5, 6, 7], rows=0),
    dict(lens=[9, 0, 0], new=[1, 0, 0], n_blocks=[77, -4, 2]),         # counts of a broken state
    dict(lens=[9, 0, 0], new=[1, 0, 0], n_free=-5),
    dict(lens=[9, 0, 0], new=[1, 0, 0], n_free=400),
    dict(lens=[0, 0, 0], new=[0, 0, 0], n_blocks=[6, 6, 6], n_free=25),  # more pages than there are
    dict(lens=[9, 9, 9], new=[9, 1, 1], free=[99] * 30, n_free=30),      # pages that do not exist
    dict(lens=[9, 9, 9], new=[9, 1, 1], n_blocks=[3, 3, 0], table=[[50, -7, 3, 1, 2, 4]] * 3),
])
def test_plan_errors_are_flagged_and_stay_inside(ops, kw):
    st = dict(pool(3, 6, 30), **{k: v for k, v in kw.items() if k in ("n_blocks", "n_free", "free", "table")})
    lens, new, rows = kw["lens"], kw["new"], kw.get("rows", 60)
    ref = plan_ref(lens, new, st["table"], st["n_blocks"], st["free"], st["n_free"], 4, rows)
    assert ref[9]
    state = [ints(st["table"]), ints(st["n_blocks"]), ints(st["free"]), ints([st["n_free"]])]
    p = ops.paged_plan(ints(lens), *state, 4, n_new=ints(new), max_rows=rows)
    check_plan(p, ref)
    # the error word collects
    word = ints([0x100])
    q = ops.paged_plan(ints(lens), *state, 4, n_new=ints(new), max_rows=rows, in_place=True, err=word)
    check_plan(q._replace(err=word ^ 0x100), ref)


def test_plan_without_requests_and_with_the_most(ops):
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    p = ops.paged_plan(e, torch.empty(0, 3, dtype=torch.int32, device="cuda"), e, ints([2, 1]), ints([2]), 4, max_rows=5)
    check_plan(p, plan_ref([], [], [], [], [2, 1], 2, 4, 5))
    B = 8192
    lens = [(b * 37) % 65 for b in range(B)]
    st = pool(B, 4, B * 4)
    p = ops.paged_plan(ints(lens), ints(st["table"]), ints(st["n_blocks"]), ints(st["free"]), ints([B * 4]), 16,
                       n_new=ints(lens), max_rows=sum(lens))
    check_plan(p, plan_ref(lens, lens, st["table"], st["n_blocks"], st["free"], B * 4, 16, sum(lens)))


def test_plan_writes_only_its_rows(ops):
    """Buffers that start and end at odd places: what lies around them stays."""
    lens, new = [9, 0, 3, 30], [2, 0, 3, 17]
    st = pool(4, 4, 16)
    for off, rows in ((0, 22), (1, 25), (2, 23), (3, 40)):
        bufs = [torch.full((64,), 77, dtype=torch.int32, device="cuda") for _ in range(4)]
        state = [torch.empty(n, dtype=torch.int32, device="cuda") for n in (5, 16, 4, 16, 1)]
        p = ops.paged_plan(ints(lens), ints(st["table"]), ints(st["n_blocks"]), ints(st["free"]), ints([16]), 8,
                           n_new=ints(new), max_rows=rows, out=[b[off:off + rows] for b in bufs] + state)
        check_plan(p._replace(block_table=p.block_table.view(4, 4)),
                   plan_ref(lens, new, st["table"], st["n_blocks"], st["free"], 16, 8, rows))
        for b in bufs:
            assert (b[:off] == 77).all() and (b[off + rows:] == 77).all()


# ----------------------------------------------------------------- append --

def rounded(x, t):
    return x.to(t)


@pytest.mark.parametrize("ti", [F32, F16, BF16])
@pytest.mark.parametrize("tc", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hk,hd,N", [(16, 16, 64, 5), (8, 2, 80, 33), (1, 1, 6, 3), (3, 1, 10, 1), (32, 8, 128, 700)])
def test_append_is_exact(ops, ti, tc, H, Hk, hd, N):
    """One f32 add and one rounding of each value: equal to torch's, bit for bit; slots that no row
    names keep what they held."""
    g = torch.Generator(device="cuda").manual_seed(N + hd)
    S = 7
    pages = -(-N // S) + 2
    qkv = torch.randn(N, (H + 2 * Hk) * hd, generator=g, device="cuda").to(ti)
    bias = torch.randn((H + 2 * Hk) * hd, generator=g, device="cuda")
    ck, cv = (torch.full((pages, S, Hk, hd), 9.0, dtype=tc, device="cuda") for _ in range(2))
    slots = torch.randperm(pages * S, generator=g, device="cuda")[:N].to(torch.int32)
    for b in (bias, None):
        q, err = ops.qkv_kv_append_paged(qkv, b, ck, cv, slots)
        x = qkv.float() + (b if b is not None else 0.0)
        qd, kd = H * hd, Hk * hd
        assert err.item() == 0 and torch.equal(q, x[:, :qd].to(ti))
        for c, part in ((ck, x[:, qd:qd + kd]), (cv, x[:, qd + kd:])):
            want = torch.full((pages * S, kd), 9.0, dtype=tc, device="cuda")
            want[slots.long()] = part.to(tc)
            assert torch.equal(c.view(pages * S, kd), want)


def test_append_skips_flags_and_keeps(ops):
    """Slot -1: the row is skipped and its q stays; a slot outside: flagged, q written, no cache row."""
    S, pages, Hk, hd = 4, 3, 2, 8
    for width in (8, 6):  # the vector kernel and the scalar one
        qd = Hk * width
        qkv = torch.randn(6, 3 * qd, device="cuda")
        ck, cv = (torch.full((pages, S, Hk, width), 5.0, device="cuda") for _ in range(2))
        q0 = torch.full((6, qd), 3.0, device="cuda")
        q, err = ops.qkv_kv_append_paged(qkv, None, ck, cv, ints([2, -1, 12, 11, -2, 2 ** 31 - 1]), q_out=q0)
        assert q.data_ptr() == q0.data_ptr() and err.item() == PAGE_OOB
        assert torch.equal(q[[0, 2, 3, 4, 5]], qkv[[0, 2, 3, 4, 5], :qd]) and (q[1] == 3.0).all()
        want = torch.full((12, qd), 5.0, device="cuda")
        want[2], want[11] = qkv[0, qd:2 * qd], qkv[3, qd:2 * qd]
        assert torch.equal(ck.view(12, qd), want)
        # without a q output, and rows that are all padding
        _, err = ops.qkv_kv_append_paged(qkv, None, ck, cv, ints([-1] * 6), with_q=False)
        assert err.item() == 0 and torch.equal(ck.view(12, qd), want)


def test_append_strided_rows_and_a_pool_of_layers(ops):
    """qkv as a slice of wider rows (aligned and not), the caches as one layer of a pool
    [pages, layers, 2, page, heads, head_dim]."""
    S, pages, L, Hk, hd, N = 4, 6, 3, 2, 16, 13
    kd = Hk * hd
    for off in (0, 8, 1):
        wide = torch.randn(N, 3 * kd + 24, device="cuda")
        qkv = wide[:, off:off + 3 * kd]
        pool_ = torch.zeros(pages, L, 2, S, Hk, hd, device="cuda", dtype=BF16)
        ck, cv = pool_[:, 1, 0], pool_[:, 1, 1]
        slots = torch.randperm(pages * S, device="cuda")[:N].to(torch.int32)
        q, err = ops.qkv_kv_append_paged(qkv, None, ck, cv, slots)
        assert err.item() == 0 and torch.equal(q, qkv[:, :kd])
        want = torch.zeros_like(pool_)
        s = slots.long()
        want[s // S, 1, 0, s % S] = qkv[:, kd:2 * kd].to(BF16).view(N, Hk, hd)
        want[s // S, 1, 1, s % S] = qkv[:, 2 * kd:].to(BF16).view(N, Hk, hd)
        assert torch.equal(pool_, want)


# -------------------------------------------------------------- attention --

def make(rows_lens, H, Hk, hd, page, qt, ct, seed, spare=2, wide=0, scale=1.0):
    """q, caches full of NaN but for the keys that are there, table, lengths."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    R, mb = len(rows_lens), max(1, -(-max(rows_lens) // page)) + wide
    have = [-(-n // page) for n in rows_lens]
    P = sum(have) + spare
    ids = torch.randperm(P, generator=g, device="cuda").to(torch.int32).tolist()
    table = [[-1] * mb for _ in range(R)]
    ck, cv = (torch.full((P, page, Hk, hd), math.nan, dtype=ct, device="cuda") for _ in range(2))
    for b, n in enumerate(rows_lens):
        for j in range(have[b]):
            table[b][j] = ids.pop()
        at = torch.arange(n, device="cuda")
        pg = ints(table[b]).long()[at // page]
        ck[pg, at % page] = (scale * torch.randn(n, Hk, hd, generator=g, device="cuda")).to(ct)
        cv[pg, at % page] = torch.randn(n, Hk, hd, generator=g, device="cuda").to(ct)
    q = torch.randn(R, H, hd, generator=g, device="cuda").to(qt)
    return q, ck, cv, ints(table), ints(rows_lens)


def check_attention(got, ref, lse=None):
    out, want_lse, bound = ref
    eps = torch.finfo(got.dtype).eps
    err = (got.double().cpu() - out).abs()
    lim = bound + eps / 2 * (out.abs() + bound) + torch.finfo(got.dtype).tiny
    assert (err <= lim).all(), (err / lim).max()
    if lse is not None:
        empty = want_lse == -math.inf
        assert torch.equal(lse.cpu() == -math.inf, empty)
        # scores as in the bound of the output (which is 2 rel |v|), then log2 and two roundings
        d = (lse.double().cpu() - want_lse).abs()[~empty]
        assert d.numel() == 0 or (d <= 1e-5 + 2.0 ** -22 * want_lse[~empty].abs()).all(), d.max()


LENS = {"edge": [1, 0, 2, 7, 8, 9, 31, 32, 33], "long": [1000, 257, 1, 4099], "one": [1537]}


@pytest.mark.parametrize("qt,ct", [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16), (BF16, F32), (F16, BF16)])
@pytest.mark.parametrize("H,Hk,hd", [(16, 16, 64), (8, 2, 128), (6, 2, 80), (5, 1, 32), (2, 1, 256), (8, 1, 8), (4, 4, 24)])
@pytest.mark.parametrize("lens", list(LENS))
def test_attention(ops, qt, ct, H, Hk, hd, lens):
    page = {"edge": 8, "long": 16, "one": 100}[lens]
    a = make(LENS[lens], H, Hk, hd, page, qt, ct, hd + H, wide=3 if lens == "edge" else 0)
    err = ints([0])
    out, lse = ops.paged_decode_attention(*a, return_lse=True, err=err)
    assert err.item() == 0
    check_attention(out, attention_ref(*a), lse)


@pytest.mark.parametrize("page", [1, 3, 64, 4096])
@pytest.mark.parametrize("H,Hk", [(4, 4), (12, 4), (7, 1), (24, 3)])
def test_attention_page_sizes_and_groups(ops, page, H, Hk):
    a = make([130, 64, 1], H, Hk, 64, page, F32, F16, page)
    check_attention(ops.paged_decode_attention(*a, scale=0.3), attention_ref(*a, scale=0.3))


def test_attention_split_over_a_long_cache(ops):
    """Few rows and many keys: the keys are split over CTAs; the same inputs give the same bits, and
    a table far wider than the lengths, or a given workspace, the same values."""
    for lens, H, Hk in (([70001], 1, 1), ([70001, 3, 0, 512], 8, 2)):
        q, ck, cv, table, n = a = make(lens, H, Hk, 64, 16, F32, BF16, 3)
        out, lse = ops.paged_decode_attention(*a, return_lse=True)
        check_attention(out, attention_ref(*a), lse)
        need = ops.paged_decode_attention_workspace(len(lens), H, Hk, 64, table.shape[1], 16, BF16)
        ws = torch.full((max(need, 16),), 255, dtype=torch.uint8, device="cuda")
        for _ in range(3):
            assert torch.equal(ops.paged_decode_attention(*a, workspace=ws), out)
        wide = torch.nn.functional.pad(table, (0, 20000), value=-1)
        check_attention(ops.paged_decode_attention(q, ck, cv, wide, n), attention_ref(*a))


def test_attention_peaked_and_flat_scores(ops):
    """Scores far apart (one key takes all, the largest first or last) and all equal."""
    q, ck, cv, table, n = a = make([900, 900, 900], 4, 2, 64, 16, F32, F32, 5, scale=12.0)
    check_attention(ops.paged_decode_attention(*a), attention_ref(*a))
    ck[:] = 0.5
    cv[torch.isnan(cv)] = 0.0
    check_attention(ops.paged_decode_attention(*a), attention_ref(*a))
    # a key with a huge score at the first and at the last place
    for at in (0, 899):
        ck.zero_()
        for b in range(3):
            ck[table[b, at // 16], at % 16] = 100.0 * q[b, 0]
        check_attention(ops.paged_decode_attention(*a), attention_ref(*a))


def test_attention_infinities_and_nan_of_real_keys(ops):
    """Inside the length the formula decides: a score of -inf weighs nothing, +inf and NaN give NaN."""
    q, ck, cv, table, n = a = make([40, 40, 40, 40], 1, 1, 64, 8, F32, F32, 6)
    q.abs_()
    ck[table[0, 2].long(), 3] = -math.inf
    ck[table[1, 2].long(), 3] = math.inf
    ck[table[2, 2].long(), 3, 0, 5] = math.nan
    cv[table[3, 2].long(), 3, 0, 5] = math.inf
    out = ops.paged_decode_attention(*a)
    keep = [j for j in range(40) if j != 19]
    k, v = (c[table[0, :5].long()].flatten(0, 1)[keep] for c in (ck, cv))
    small = (q[:1], k[None, :, :, :].contiguous(), v[None].contiguous(), ints([[0]]), ints([39]))
    check_attention(out[:1], attention_ref(*small))
    assert out[1].isnan().all() and out[2].isnan().all()
    assert out[3, 0, 5] == math.inf and out[3, 0, :5].isfinite().all()


@pytest.mark.parametrize("qt,ct,H,Hk", [(F32, F32, 2, 1), (F16, F16, 8, 2), (BF16, BF16, 2, 2), (F32, F32, 8, 1)])
def test_attention_scores_of_minus_infinity(ops, qt, ct, H, Hk):
    """Whole tiles of keys whose score is -inf weigh nothing; where all are, the row counts as empty."""
    q, ck, cv, table, n = make([700, 700, 90], H, Hk, 64, 16, qt, ct, 11)
    q.abs_().clamp_(min=0.01)
    gone = torch.zeros(700, dtype=torch.bool)
    gone[:300], gone[310:690] = True, True
    for b, mask in ((0, gone), (2, torch.ones(90, dtype=torch.bool))):
        at = torch.arange(len(mask), device="cuda")[mask.cuda()]
        ck[table[b].long()[at // 16], at % 16] = -math.inf
    out, lse = ops.paged_decode_attention(q, ck, cv, table, n, return_lse=True)
    left = torch.arange(700, device="cuda")[~gone.cuda()]
    k, v = (c[table[0].long()[left // 16], left % 16][None].contiguous() for c in (ck, cv))
    check_attention(out[:1], attention_ref(q[:1], k, v, ints([[0]]), ints([len(left)])), lse[:1])
    check_attention(out[1:2], attention_ref(q[1:2], ck, cv, table[1:2], n[1:2]), lse[1:2])
    assert not out[2].any() and (lse[2] == -math.inf).all()


@pytest.mark.parametrize("H,Hk,hd", [(3, 1, 24), (8, 2, 32), (12, 1, 40), (16, 2, 64), (17, 1, 96), (4, 1, 128)])
@pytest.mark.parametrize("qt", [F32, BF16])
@pytest.mark.parametrize("kpow,vpow", [(0, 0), (60, -100), (-60, 110)])
def test_attention_f32_caches_of_any_magnitude(ops, H, Hk, hd, qt, kpow, vpow):
    """Keys and values far from 1, scores of a like size (300 values of 2^110 sum to less than 2^128)."""
    q, ck, cv, table, n = make([300, 33, 1], H, Hk, hd, 16, qt, F32, hd)
    q, ck = (q.float() * 2.0 ** -kpow).to(qt), ck * 2.0 ** kpow
    cv = cv.clamp(-0.9, 0.9) * 2.0 ** vpow
    a = (q, ck, cv, table, n)
    check_attention(ops.paged_decode_attention(*a), attention_ref(*a))


@pytest.mark.parametrize("ct,H,Hk,hd", [(F32, 4, 1, 32), (F32, 6, 2, 64), (F32, 3, 1, 80), (F32, 9, 1, 128), (BF16, 4, 1, 80)])
def test_attention_infinite_keys_and_bad_pages_of_grouped_heads(ops, ct, H, Hk, hd):
    """Keys of -inf under a positive query, and pages outside the cache, in one row: both weigh nothing."""
    q, ck, cv, table, n = make([200, 47, 16], H, Hk, hd, 16, BF16 if ct == BF16 else F32, ct, hd)
    q.abs_().clamp_(min=0.01)
    at = torch.arange(200, device="cuda")
    gone = (at < 3) | (at >= 64) & (at < 96) | (at == 150)
    ck[table[0].long()[at[gone] // 16], at[gone] % 16] = -math.inf
    bad = table.clone()
    bad[0, 2], bad[0, 7], bad[2, 0] = -1, ck.shape[0], 2 ** 31 - 1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = ops.paged_decode_attention(q, ck, cv, bad, n, err=err)
    assert err.item() == PAGE_OOB and not out[2].any()
    left = at[~gone & (at // 16 != 2) & (at // 16 != 7)]
    k, v = (c[table[0].long()[left // 16], left % 16][None].contiguous() for c in (ck, cv))
    check_attention(out[:1], attention_ref(q[:1], k, v, ints([[0]]), ints([len(left)])))
    check_attention(out[1:2], attention_ref(q[1:2], ck, cv, table[1:2], n[1:2]))


def test_attention_many_rows_of_one_request(ops):
    """row_reqs: the tokens of a prefill chunk, each row with its own length, and unordered requests."""
    q, ck, cv, table, n = make([50, 20, 33], 4, 2, 64, 16, F32, F16, 7)
    reqs = [0] * 50 + [2, 1, 2, 1]
    lens = list(range(1, 51)) + [33, 20, 1, 0]
    q = torch.randn(len(reqs), 4, 64, device="cuda")
    out, lse = ops.paged_decode_attention(q, ck, cv, table, ints(lens), row_reqs=ints(reqs), return_lse=True)
    check_attention(out, attention_ref(q, ck, cv, table, ints(lens), ints(reqs)), lse)


def test_attention_of_more_rows_than_a_grid_dimension_holds(ops):
    """The rows of a large prefill: 70,000, most of them equal, checked against a few."""
    q, ck, cv, table, n = make([9, 4], 4, 2, 32, 4, F32, F16, 12)
    N = 70000
    r = torch.arange(N, device="cuda")
    reqs, lens = (r % 2).to(torch.int32), (1 + r % 4).to(torch.int32)
    out = ops.paged_decode_attention(q[r % 2].contiguous(), ck, cv, table, lens, row_reqs=reqs)
    check_attention(out[:4], attention_ref(q[r[:4] % 2], ck, cv, table, lens[:4], reqs[:4]))
    assert torch.equal(out, out[:4].repeat(N // 4, 1, 1))


def test_attention_bad_indexes_are_left_out(ops):
    q, ck, cv, table, n = make([40, 40, 40, 40], 2, 1, 64, 8, F32, F32, 8)
    bad = table.clone()
    bad[0, 1], bad[1, 4], bad[1, 0] = -1, ck.shape[0], 2 ** 31 - 1
    err = ints([0])
    out, lse = ops.paged_decode_attention(q, ck, cv, bad, n, return_lse=True, err=err)
    assert err.item() == PAGE_OOB
    check_attention(out, attention_ref(q, ck, cv, bad, n), lse)
    err.zero_()
    reqs, lens = ints([3, -1, 4, 0]), ints([40, 40, 40, -2])
    out = ops.paged_decode_attention(q, ck, cv, table, lens, row_reqs=reqs, err=err)
    assert err.item() == PAGE_OOB | LENGTH and not out[1:].any()
    check_attention(out[:1], attention_ref(q[:1], ck, cv, table, lens[:1], reqs[:1]))
    err.zero_()
    full = ops.paged_decode_attention(q, ck, cv, table, n, err=err)
    over = ops.paged_decode_attention(q, ck, cv, table, ints([41, 40, 2 ** 31 - 1, 40]), err=err)
    assert err.item() == LENGTH and torch.equal(full, over)
    err.zero_()
    gone = torch.full_like(table, -1)  # nothing left: zeros
    out, lse = ops.paged_decode_attention(q, ck, cv, gone, n, return_lse=True, err=err)
    assert err.item() == PAGE_OOB and not out.any() and (lse == -math.inf).all()


def test_attention_strided_q_a_pool_of_layers_and_out(ops):
    """q as a slice of the QKV rows, the caches as one layer of a pool, the output given."""
    q, ck, cv, table, n = make([100, 37], 4, 2, 64, 16, F32, BF16, 9)
    pool_ = torch.full((ck.shape[0], 3, 2, *ck.shape[1:]), math.nan, dtype=BF16, device="cuda")
    pool_[:, 1, 0], pool_[:, 1, 1] = ck, cv
    for off in (0, 4, 1):
        wide = torch.full((2, 4 * 64 + 24), math.nan, device="cuda")
        wide[:, off:off + 256] = q.view(2, 256)
        qs = wide[:, off:off + 256].unflatten(1, (4, 64))
        out = torch.full((2, 4, 64), 7.0, device="cuda")
        got = ops.paged_decode_attention(qs, pool_[:, 1, 0], pool_[:, 1, 1], table, n, out=out)
        assert got.data_ptr() == out.data_ptr()
        check_attention(got, attention_ref(q, ck, cv, table, n))


def test_append_and_attention_past_32_bit_offsets(ops):
    """A cache of more than 2^32 bytes and 2^31 elements: its last pages."""
    Hk, hd, S = 8, 128, 64
    P = (1 << 31) // (Hk * hd * S) + 3
    ck = torch.empty(P, S, Hk, hd, dtype=F16, device="cuda")
    cv = torch.empty(P, S, Hk, hd, dtype=F16, device="cuda")
    table, n = ints([[P - 1, 0, P - 2]]), ints([150])
    rows = torch.randn(150, 3 * Hk * hd, device="cuda")
    j = torch.arange(150, device="cuda")
    slots = (table[0].long()[j // S] * S + j % S).to(torch.int32)
    q, err = ops.qkv_kv_append_paged(rows, None, ck, cv, slots)
    assert err.item() == 0
    small_k, small_v = ck[table[0].long()], cv[table[0].long()]
    assert torch.equal(small_k.flatten(0, 1)[:150], rows[:, Hk * hd:2 * Hk * hd].half().view(150, Hk, hd))
    small_k.flatten(0, 1)[150:] = 0
    small_v.flatten(0, 1)[150:] = 0
    out = ops.paged_decode_attention(q[-1:].view(1, Hk, hd), ck, cv, table, n)
    check_attention(out, attention_ref(q[-1:].view(1, Hk, hd), small_k, small_v, ints([[0, 1, 2]]), n))


def test_a_step_replayed_from_a_graph_and_on_another_stream(ops):
    """plan -> append -> attention captured once; replays follow the lengths in device memory, and two
    captured steps that run at the same time do not disturb one another."""
    B, page, ctx, Hk, hd = 5, 8, 3000, 2, 64
    mb = -(-ctx // page)
    P = B * mb

    def state():
        s = dict(lens=ints([0] * B), qkv=torch.zeros(B, 3 * Hk * hd, device="cuda"),
                 ck=torch.full((P, page, Hk, hd), math.nan, device="cuda", dtype=F16), table=ints([[-1] * mb] * B),
                 n_blocks=ints([0] * B), free=ints(list(range(P))), n_free=ints([P]), err=ints([0]))
        s["cv"] = s["ck"].clone()
        return s

    def step(s):
        p = ops.paged_plan(s["lens"], s["table"], s["n_blocks"], s["free"], s["n_free"], page, in_place=True, err=s["err"])
        q, _ = ops.qkv_kv_append_paged(s["qkv"], None, s["ck"], s["cv"], p.slots, err=s["err"])
        return ops.paged_decode_attention(q.view(B, Hk, hd), s["ck"], s["cv"], p.block_table, p.row_lens,
                                          row_reqs=p.row_reqs, err=s["err"])

    runs = []
    for k in range(2):
        s = state()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(s)  # warm-up (lengths are zero: nothing is written)
        torch.cuda.current_stream().wait_stream(stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s["out"] = step(s)
        runs.append((s, g, stream))
    twin = [state() for _ in range(2)]
    gen = torch.Generator(device="cuda").manual_seed(1)
    lens = [0] * B
    for t in range(30):
        lens = [n + 1 for n in lens] if t != 20 else [0, *(n + 1 for n in lens[1:])]
        qkv = torch.randn(2, B, 3 * Hk * hd, generator=gen, device="cuda")
        torch.cuda.synchronize()
        for k, (s, g, stream) in enumerate(runs):
            with torch.cuda.stream(stream):
                s["lens"].copy_(ints(lens))
                s["qkv"].copy_(qkv[k])
                g.replay()
        torch.cuda.synchronize()
        for k, (s, _, _) in enumerate(runs):
            twin[k]["lens"].copy_(ints(lens))
            twin[k]["qkv"].copy_(qkv[k])
            assert torch.equal(step(twin[k]), s["out"]), (t, k)
            assert s["err"].item() == twin[k]["err"].item() == 0
    for k, (s, _, _) in enumerate(runs):
        n = ints(lens)
        if 0 in lens:
            continue
        q = s["qkv"][:, :Hk * hd].view(B, Hk, hd)
        check_attention(s["out"], attention_ref(q, s["ck"], s["cv"], s["table"], n))
    del runs


@pytest.mark.parametrize("qt,ct", [(F16, F16), (F32, F16), (BF16, F16), (F32, BF16), (BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("H,Hk,hd", [(4, 4, 64), (4, 2, 64), (16, 2, 32), (12, 4, 80), (8, 1, 128)])
@pytest.mark.parametrize("nats", [12, 14, 16, 18, 24])
def test_attention_of_a_key_that_takes_the_weight_and_holds_nothing(ops, qt, ct, H, Hk, hd, nats):
    """One key whose value is zero, all others `nats` below it: the result is what the others' small
    probabilities sum to.  The bound is relative to them, as the formula in f32 is."""
    lens = [2049, 40, 20000]
    _, ck, cv, table, n = make(lens, H, Hk, hd, 16, qt, ct, hd + nats)
    g = torch.Generator(device="cuda").manual_seed(nats)
    q = torch.ones(3, H, hd, device="cuda", dtype=qt)
    for b, m in enumerate(lens):
        at = torch.arange(m, device="cuda")
        pg = table[b].long()[at // 16]
        # scores are sqrt(hd) times these: the sink's 0
        low = -nats / hd ** 0.5 + 0.02 * torch.randn(m, Hk, 1, generator=g, device="cuda")
        low[m // 3] = 0.0
        ck[pg, at % 16] = low.expand(m, Hk, hd).to(ct)
        v = 500.0 + 1000.0 * torch.rand(m, Hk, hd, generator=g, device="cuda")
        v[m // 3] = 0.0
        cv[pg, at % 16] = v.to(ct)
    a = (q, ck, cv, table, n)
    out, lse = ops.paged_decode_attention(*a, return_lse=True)
    check_attention(out, attention_ref(*a), lse)


@pytest.mark.parametrize("ct,H", [(F16, 2), (BF16, 2), (F16, 8), (BF16, 8), (F32, 2), (F32, 8)])
def test_attention_long_sums_do_not_drift(ops, ct, H):
    """65,536 keys in one CTA (so many rows that the keys are not split), equal scores, values of one sign:
    the mean of the values.  The weights are 1 and their sum exact.  A warp has 16,384 keys and adds tiles of
    8 or more: at most N = 2048 f32 additions, each relative to a partial sum.  Rounded to nearest, their
    errors are independent of sign with a variance of at most u^2 / 3 (u = 2^-24), together
    u sqrt(sum (i / N)^2 / 3) = u sqrt(N / 9) = 15 u; six of them: 91 u.  Within a tile at most 17 terms lose
    2^-23 of the largest, 1, against a sum of 8 * 0.5 or more: 9 u; joins and the quotient 10 u.  Additions
    that truncate would be off by N / 4 2^-23 = 1024 u."""
    n, S, hd, R = 65536, 64, 64, 5000
    g = torch.Generator(device="cuda").manual_seed(H)
    ck = torch.randn(1, 1, 1, hd, generator=g, device="cuda").to(ct).expand(n // S, S, 1, hd).contiguous()
    cv = (0.5 + 0.5 * torch.rand(n // S, S, 1, hd, generator=g, device="cuda")).to(ct)
    table = torch.randperm(n // S, generator=g, device="cuda").to(torch.int32)[None]
    q = torch.randn(R, H, hd, generator=g, device="cuda")
    lens = torch.zeros(R, dtype=torch.int32, device="cuda")
    lens[17] = n
    assert ops.paged_decode_attention_workspace(R, H, 1, hd, n // S, S, ct) == 0
    out = ops.paged_decode_attention(q, ck, cv, table, lens, row_reqs=torch.zeros_like(lens))
    want = cv.double().mean((0, 1, 2))
    off = (out[17].double() / want - 1).abs().max().item() * 2.0 ** 24
    assert off < 91 + 9 + 10, off
    assert not out[:17].any() and not out[18:].any()


@pytest.mark.parametrize("ct,H", [(F16, 2), (BF16, 2), (F16, 8), (BF16, 8), (F32, 2), (F32, 8)])
def test_attention_long_weighted_sums_do_not_drift(ops, ct, H):
    """The same with weights of all sizes around 1 (scores with a deviation of a half), which the values'
    few bits do not make exact: 91 u for the sums as above; the sum of the weights, 2048 additions a lane,
    the same averaged over the 4 lanes: 46 u; a tile's sum is a quarter of 16 times its largest term or more:
    20 u; e^ 8 u; the terms of q 4 u (the scores' own errors have either sign and average out); joins and the
    quotient 10 u."""
    n, S, hd, R = 65536, 64, 64, 5000
    g = torch.Generator(device="cuda").manual_seed(H)
    ck = (0.5 * torch.randn(n // S, S, 1, hd, generator=g, device="cuda")).to(ct)
    cv = (0.5 + 0.5 * torch.rand(n // S, S, 1, hd, generator=g, device="cuda")).to(ct)
    table = torch.randperm(n // S, generator=g, device="cuda").to(torch.int32)[None]
    q = torch.randn(R, H, hd, generator=g, device="cuda")
    lens = torch.zeros(R, dtype=torch.int32, device="cuda")
    lens[17] = n
    out = ops.paged_decode_attention(q, ck, cv, table, lens, row_reqs=torch.zeros_like(lens))
    k, v = (c[table[0].long()].flatten(0, 2).double() for c in (ck, cv))
    want = torch.softmax(q[17].double() @ k.T / hd ** 0.5, -1) @ v
    off = (out[17].double() / want - 1).abs().max().item() * 2.0 ** 24
    assert off < 91 + 46 + 20 + 8 + 4 + 10, off


@pytest.mark.parametrize("qt,ct,H,Hk", [(F32, F16, 8, 2), (F32, BF16, 8, 1), (BF16, F16, 4, 2), (F16, BF16, 2, 1), (F16, F32, 3, 1)])
def test_attention_scores_of_minus_infinity_with_q_of_another_type(ops, qt, ct, H, Hk):
    """The same where the tensor cores take q in several terms, some of them 0."""
    test_attention_scores_of_minus_infinity(ops, qt, ct, H, Hk)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("table", [[[7, 1, 2, -1], [-3, 4, 5, -1], [6, 3, 0, -1]], [[7, 1, 2, -1], [8, 4, 99, -1], [6, 3, 0, -1]],
                                   [[2 ** 31 - 1, 1, 2, -1], [8, 4, 9, -1], [6, 3, 0, -1]]])
def test_plan_flags_bad_pages_that_a_request_keeps(ops, in_place, table):
    """A page outside the pool in a block that none of the step's rows lies in: flagged, in place or not."""
    lens, new, have = [9, 12, 0], [1, 0, 0], [3, 3, 0]
    free = [10, 11, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0]
    ref = plan_ref(lens, new, table, have, free, 2, 4, 4)
    assert ref[9] == PAGE_OOB
    p = ops.paged_plan(ints(lens), ints(table), ints(have), ints(free), ints([2]), 4, n_new=ints(new), max_rows=4,
                       in_place=in_place)
    check_plan(p, ref)


@pytest.mark.parametrize("qt,ct", [(F32, F32), (BF16, F32), (F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("H,Hk,hd", [(3, 1, 136), (10, 2, 160), (7, 1, 208), (6, 2, 216), (5, 1, 248), (8, 2, 256)])
@pytest.mark.parametrize("lens", list(LENS))
def test_attention_grouped_heads_of_more_than_128_elements(ops, qt, ct, H, Hk, hd, lens):
    """Both kernels for them (f32: up to 208 elements, and above), with chunks of four heads that are not full."""
    a = make(LENS[lens], H, Hk, hd, 16, qt, ct, hd + H)
    out, lse = ops.paged_decode_attention(*a, return_lse=True)
    check_attention(out, attention_ref(*a), lse)
    if lens == "edge":  # unsplit, rows of all lengths
        many = torch.randn(300, H, hd, device="cuda").to(qt)
        reqs = torch.arange(300, device="cuda", dtype=torch.int32) % len(LENS[lens])
        n = a[4][reqs.long()].contiguous()
        got = ops.paged_decode_attention(many, *a[1:4], n, row_reqs=reqs)
        check_attention(got, attention_ref(many, *a[1:4], n, reqs))


@pytest.mark.parametrize("scale", [0.0, -0.5, 1e-30, 3.0])
@pytest.mark.parametrize("qt,ct,H,Hk", [(F32, F32, 2, 1), (F32, F32, 8, 2), (F32, F16, 4, 1), (F32, BF16, 8, 2), (F16, F16, 4, 4), (BF16, BF16, 4, 1)])
def test_attention_of_any_scale(ops, qt, ct, H, Hk, scale):
    a = make([700, 33, 0, 1], H, Hk, 64, 16, qt, ct, 5)
    out, lse = ops.paged_decode_attention(*a, scale=scale, return_lse=True)
    # the reference's bound takes the scale as |scale|: its sign goes to q, which is exact
    ref = attention_ref(math.copysign(1.0, scale) * a[0], *a[1:], scale=abs(scale))
    check_attention(out, ref, lse)


def test_plan_in_place_with_the_most_requests(ops):
    B = 8192
    lens = [(b * 37) % 65 for b in range(B)]
    st = pool(B, 4, B * 4)
    p = ops.paged_plan(ints(lens), ints(st["table"]), ints(st["n_blocks"]), ints(st["free"]), ints([B * 4]), 16,
                       n_new=ints(lens), max_rows=sum(lens), in_place=True)
    ref = plan_ref(lens, lens, st["table"], st["n_blocks"], st["free"], B * 4, 16, sum(lens))
    check_plan(p, ref)
    cut = [n // 2 for n in lens]
    p = ops.paged_plan(ints(cut), p.block_table, p.n_blocks, p.free_list, p.n_free, 16, n_new=ints([0] * B), max_rows=0,
                       in_place=True)
    check_plan(p, plan_ref(cut, [0] * B, ref[5], ref[6], ref[7], ref[8], 16, 0))


def test_attention_split_calls_at_the_same_time_and_replayed(ops):
    """Two captured calls that split a long cache over the workspace, each with its own, replayed on two
    streams while their lengths change: what the eager calls give."""
    calls = []
    for k in range(2):
        q, ck, cv, table, n = make([30001], 2, 1, 64, 16, F32, BF16, 20 + k)
        need = ops.paged_decode_attention_workspace(1, 2, 1, 64, table.shape[1], 16, BF16)
        assert need > 0
        ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
        args = (q, ck, cv, table, n)
        ops.paged_decode_attention(*args, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.paged_decode_attention(*args, workspace=ws)
        calls.append((args, g, out, torch.cuda.Stream()))
    for lens in ((30001, 30001), (1, 29000), (0, 17), (257, 4096), (30001, 2)):
        for (args, g, out, s), n in zip(calls, lens):
            args[4].fill_(n)
        torch.cuda.synchronize()
        for _ in range(3):
            for args, g, out, s in calls:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for args, g, out, s in calls:
            assert torch.equal(out, ops.paged_decode_attention(*args))
            check_attention(out, attention_ref(*args))
    del calls
