"""cbx_token_logprobs on the GPU against the definition in 64 bits (ids
exactly; values with the bounds that tests/_paged.py derives)."""
import math

import pytest

torch = pytest.importorskip("torch")

from _paged import TOKEN_OOB, logprobs_ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from chatterbox_amdvulkan_b200 import ops as _ops
    return _ops


def check(got, x, tokens, k):
    lp, ent, ids, top, rel, ent_tol = logprobs_ref(x, tokens, k)
    assert torch.equal(got.top_ids.cpu(), ids)
    u = 2.0 ** -24
    for g, w, tol in ((got.logprobs, lp, None), (got.top_logprobs, top, None), (got.entropy, ent, ent_tol)):
        if g is None or not w.numel():
            continue
        g = g.double().cpu()
        tol = (rel + 4 * u * w.abs()) if tol is None else tol
        inf = w == -math.inf
        assert torch.equal(g == -math.inf, inf)
        d = (g - w).abs()[~inf]
        assert (d <= tol[~inf]).all(), (d / tol[~inf]).max()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("N,V", [(1, 6563), (3, 1), (5, 2), (4, 7), (9, 33), (300, 257), (7, 50276), (2, 131073)])
@pytest.mark.parametrize("k", [0, 1, 5, 32])
def test_logprobs(ops, t, N, V, k):
    g = torch.Generator(device="cuda").manual_seed(V + k)
    x = (3.0 * torch.randn(N, V, generator=g, device="cuda")).to(t)
    tokens = torch.randint(0, V, (N,), generator=g, device="cuda", dtype=torch.int32)
    got = ops.token_logprobs(x, tokens, top_k=min(k, V))
    assert got.err.item() == 0
    check(got, x, tokens, min(k, V))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [1, 2, 300, 6563])
def test_logprobs_of_one_sure_token(ops, t, V):
    """One token takes all: its log probability is 0 up to rounding and never above, the entropy never below."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(2000, V, generator=g, device="cuda")
    tokens = torch.randint(0, V, (2000,), generator=g, device="cuda", dtype=torch.int32)
    x.scatter_(1, tokens.long()[:, None], x.gather(1, tokens.long()[:, None]) + 40.0 * (V > 1))
    x = x.to(t)
    got = ops.token_logprobs(x, tokens, top_k=1)
    check(got, x, tokens, 1)
    assert (got.logprobs <= 0).all() and (got.top_logprobs <= 0).all() and (got.entropy >= 0).all()


@pytest.mark.parametrize("t", TYPES)
def test_logprobs_strided_and_shifted_rows(ops, t):
    """Rows that start at every place within 16 bytes; a padded vocabulary whose tail must not count."""
    for off in range(9):
        wide = torch.randn(6, 1000, device="cuda").to(t)
        wide[:, off + 805:] = 100.0
        wide[:, :off] = 100.0
        x = wide[:, off:off + 805]
        tokens = torch.randint(0, 805, (6,), device="cuda", dtype=torch.int32)
        check(ops.token_logprobs(x, tokens, top_k=7), x, tokens, 7)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [37, 2048, 6563])
def test_logprobs_ties(ops, t, V):
    """Equal logits go by their index: all equal, few values, signed zeros, the largest last."""
    g = torch.Generator(device="cuda").manual_seed(V)
    rows = [torch.zeros(V, device="cuda"), torch.randint(0, 3, (V,), generator=g, device="cuda").float(),
            torch.where(torch.rand(V, generator=g, device="cuda") < 0.5, 0.0, -0.0),
            torch.arange(V, device="cuda").float().floor_divide(8), -torch.arange(V, device="cuda").float().floor_divide(8),
            torch.full((V,), -7.5, device="cuda")]
    x = torch.stack(rows).to(t)
    tokens = torch.randint(0, V, (len(rows),), generator=g, device="cuda", dtype=torch.int32)
    for k in (1, 4, 32):
        check(ops.token_logprobs(x, tokens, top_k=k), x, tokens, k)


@pytest.mark.parametrize("V", [6563, 50276])
def test_logprobs_large_ones_together(ops, V):
    """The largest logits lie side by side, in one stride of the threads, or all over in rising order:
    the choice of alternatives does not depend on where they are."""
    base = torch.randn(6, V, device="cuda")
    base[0, 100:140] += 30
    base[1, ::256] += 30
    base[2, ::2048] += 30
    base[3] = torch.arange(V, device="cuda") * 1e-3
    base[4] = -torch.arange(V, device="cuda") * 1e-3
    base[5, :4096] += 30
    for t in (torch.float32, torch.float16):
        x = base.to(t)
        tokens = torch.arange(6, device="cuda", dtype=torch.int32)
        for k in (20, 32):
            check(ops.token_logprobs(x, tokens, top_k=k), x, tokens, k)


@pytest.mark.parametrize("t", TYPES)
def test_logprobs_masked_rows(ops, t):
    """-inf and the type's lowest value as masks: most of a row, all but one, and a far offset."""
    V = 1000
    low = torch.finfo(t).min
    x = torch.randn(6, V, device="cuda").to(t)
    x[0, 3:] = -math.inf
    x[1, :999] = -math.inf
    x[2, ::2] = -math.inf
    x[3, 5:] = low
    x[4] = low                     # uniform
    x[5] += 200.0
    tokens = torch.tensor([1, 999, 2, 700, 3, 9], dtype=torch.int32, device="cuda")
    got = ops.token_logprobs(x, tokens, top_k=5)
    check(got, x, tokens, 5)
    assert got.logprobs[2] == -math.inf and abs(got.logprobs[4].item() + math.log(V)) < 1e-5


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [50, 1000, 6563])
def test_logprobs_largest_near_the_types_lowest(ops, t, V):
    """Rows whose largest logit is itself a mask value, beside -inf and other mask values."""
    low = torch.finfo(t).min
    x = torch.full((5, V), -math.inf, device="cuda", dtype=t)
    x[0, ::3] = low
    x[1] = low
    x[2, 1::2] = -1e30 if t != torch.float16 else -65000.0
    x[3, ::2], x[3, 5] = low, low / 2
    x[4], x[4, 7] = -60000.0, 3.0
    tokens = torch.tensor([3, 5, 1, 5, 7], dtype=torch.int32, device="cuda")
    for k in (1, 6):
        check(ops.token_logprobs(x, tokens, top_k=k), x, tokens, k)


def test_logprobs_rows_without_a_distribution(ops):
    """Nothing but -inf, a +inf, a NaN: values NaN; the order of the alternatives still holds."""
    x = torch.randn(4, 500, device="cuda")
    x[0] = -math.inf
    x[1, 44] = math.inf
    x[2, 45], x[2, 400] = math.nan, math.nan
    tokens = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    got = ops.token_logprobs(x, tokens, top_k=3)
    assert got.logprobs[:3].isnan().all() and got.entropy[:3].isnan().all() and got.top_logprobs[:3].isnan().all()
    assert got.top_ids[0].tolist() == [0, 1, 2] and got.top_ids[1, 0] == 44 and got.top_ids[2, :2].tolist() == [45, 400]
    check(ops.token_logprobs(x[3:], tokens[3:], top_k=3), x[3:], tokens[3:], 3)
    assert got.logprobs[3].isfinite()


def test_logprobs_tokens_outside(ops):
    x = torch.randn(4, 100, device="cuda")
    tokens = torch.tensor([5, -1, 99, 3], dtype=torch.int32, device="cuda")
    got = ops.token_logprobs(x, tokens)
    assert got.err.item() == 0 and got.logprobs[1].isnan() and got.logprobs[[0, 2, 3]].isfinite().all()
    for bad in (100, -2, 2 ** 31 - 1):
        tokens[3] = bad
        got = ops.token_logprobs(x, tokens)
        assert got.err.item() == TOKEN_OOB and got.logprobs[3].isnan() and got.entropy.isfinite().all()
    got = ops.token_logprobs(x, None, top_k=2)
    assert got.logprobs is None
    check(got, x, None, 2)
    assert ops.token_logprobs(x[:0], None).entropy.numel() == 0


def test_logprobs_twice_the_same_and_replayed(ops):
    x = torch.randn(500, 6563, device="cuda").bfloat16()
    tokens = torch.randint(0, 6563, (500,), device="cuda", dtype=torch.int32)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    first = ops.token_logprobs(x, tokens, top_k=8, err=err)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        second = ops.token_logprobs(x, tokens, top_k=8, err=err)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        third = ops.token_logprobs(x, tokens, top_k=8, err=err)
    g.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first[:4], second[:4], third[:4]):
        assert torch.equal(a, b) and torch.equal(a, c)
    x.neg_()
    g.replay()
    torch.cuda.synchronize()
    check(third, x, tokens, 8)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [3, 50, 1000, 6563])
def test_logprobs_of_any_magnitude(ops, t, V):
    """Rows of one value from 10^3 to the type's largest power of ten, both signs; rows of a few neighbours of
    that value; and finite masks of that size around logits of ordinary size."""
    g = torch.Generator(device="cuda").manual_seed(V)
    last = 4 if t == torch.float16 else 37
    size = 10.0 ** torch.arange(3, last + 1, device="cuda", dtype=torch.float64).repeat_interleave(2)
    size = size * torch.tensor([1.0, -1.0], device="cuda").repeat(len(size) // 2)
    far = size[:, None].expand(-1, V)
    # the neighbours: up to 8 steps of the type above the value
    step = torch.finfo(t).eps * size.abs()[:, None]
    near = far + step * torch.randint(0, 9, far.shape, generator=g, device="cuda")
    masked = torch.where(torch.rand(far.shape, generator=g, device="cuda") < 0.7, -far.abs(), torch.randn(far.shape, generator=g, device="cuda").double())
    x = torch.cat([far, near, masked]).to(t)
    tokens = torch.randint(0, V, (len(x),), generator=g, device="cuda", dtype=torch.int32)
    k = min(V, 4)
    check(ops.token_logprobs(x, tokens, top_k=k), x, tokens, k)
    check(ops.token_logprobs(x, tokens), x, tokens, 0)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [300, 6563])
def test_logprobs_beside_large_finite_masks(ops, t, V):
    """Logits of ordinary size in the last places of a row whose rest is one large value: whole threads see
    nothing but the mask.  (x log2 e of the odd ones is 122 to 126 above its rounded value.)"""
    masks = [-2785017856.0, -3998240768.0, -1e12, -1e30, -65504.0, torch.finfo(t).min]
    x = torch.tensor(masks, device="cuda")[:, None].repeat(1, V)
    g = torch.Generator(device="cuda").manual_seed(V)
    x[:, -40:] = torch.randn(len(masks), 40, generator=g, device="cuda")
    x = x.to(t)
    tokens = torch.tensor([V - 1, V - 7, 0, V - 40, 5, V - 2], device="cuda", dtype=torch.int32)
    for k in (0, 5):
        check(ops.token_logprobs(x, tokens, top_k=k), x, tokens, k)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [40, 130, 6563, 50276])
def test_logprobs_of_half_masked_vocabularies(ops, t, V):
    """-inf over whole threads: the first half, the last half, all but the last place, every block but one."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = 3.0 * torch.randn(4, V, generator=g, device="cuda")
    x[0, :V // 2] = -math.inf
    x[1, V // 2:] = -math.inf
    x[2, :-1] = -math.inf
    x[3, :V // 3], x[3, V // 3 + 9:] = -math.inf, -math.inf
    x = torch.cat([x, x - 1000.0]).to(t)
    tokens = torch.tensor([V - 1, 0, V - 1, V // 3] * 2, dtype=torch.int32, device="cuda")
    for k in (0, 3):
        check(ops.token_logprobs(x, tokens, top_k=k), x, tokens, k)
