"""The paged T3 step (chatterbox_amdvulkan_b200/decode_step.py, T3PagedDecode):
plan, gather, QKV epilogue, attention and log probabilities as a server runs
them, against the same model in plain torch on whole sequences."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from chatterbox_amdvulkan_b200 import decode_step
    torch.backends.cuda.matmul.allow_tf32 = False
    return decode_step


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def whole(m, ids):
    """Final hidden states of one whole sequence in f64, K and V rounded to the cache's type."""
    d = lambda t: t.double()  # noqa: E731
    n, hd = len(ids), m.D // m.H
    h = d(m.tok_emb)[ids] + d(m.pos_emb)[:n]
    causal = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    ln = torch.nn.functional.layer_norm
    for P in m.layers:
        y = ln(h, (m.D,), d(P["ln1_w"]), d(P["ln1_b"]), m.eps)
        q, k, v = (y @ d(P["qkv_w"]) + d(P["qkv_b"])).split(m.D, -1)
        k, v = (t.float().to(m.cache_k.dtype).double() for t in (k, v))
        q, k, v = (t.view(n, m.H, hd).transpose(0, 1) for t in (q, k, v))
        s = (q @ k.transpose(1, 2) / hd ** 0.5).masked_fill(~causal, float("-inf"))
        a = (torch.softmax(s, -1) @ v).transpose(0, 1).reshape(n, m.D)
        r = a @ d(P["out_w"]) + d(P["out_b"]) + h
        y = ln(r, (m.D,), d(P["ln2_w"]), d(P["ln2_b"]), m.eps)
        f = torch.nn.functional.gelu(y @ d(P["fc_w"]) + d(P["fc_b"]), approximate="tanh")
        h = f @ d(P["proj_w"]) + d(P["proj_b"]) + r
    return ln(h, (m.D,), d(m.lnf_w), d(m.lnf_b), m.eps)


@pytest.mark.parametrize("cache_dtype", [torch.float32, torch.bfloat16])
def test_a_servers_requests_match_whole_sequences(dec, cache_dtype):
    """Requests start at different steps with prompts of unequal length, decode side by side, are fed
    several tokens at a time, end and hand their pages on.  Every row's hidden state equals that of
    the whole sequence.  Bounds, relative to the largest value: sums of up to 4096 products in f32 are
    off by about sqrt(4096) 2^-24 = 4e-6 each, 4 GEMMs in each of 3 layers: 5e-5; taken twice.  With
    a bf16 cache a difference of that size upstream can round a K or V value the other way (2^-8 of
    it), as in the slab step's test."""
    tol = 1e-4 if cache_dtype == torch.float32 else 4e-3
    m = dec.T3PagedDecode(3, max_reqs=4, n_pages=24, page_size=8, max_context=100, D=256, H=4, F=1024,
                          vocab=500, cache_dtype=cache_dtype, seed=5)
    g = torch.Generator().manual_seed(6)
    seqs = {}  # request -> ids so far
    #        per step: request -> tokens fed (0: it ends)
    script = [{0: 37, 1: 1}, {0: 1, 1: 1, 2: 60}, {0: 1, 1: 5, 2: 1}, {0: 0, 1: 1, 2: 1, 3: 3},
              {0: 64, 1: 1, 2: 0, 3: 1}, {0: 1, 1: 1, 2: 9, 3: 30}]
    for fed in script:
        lens, new, rows, want = [0] * 4, [0] * 4, [], []
        for b in range(4):
            if fed.get(b, 0) == 0:
                seqs.pop(b, None)
                continue
            ids = torch.randint(0, 500, (fed[b],), generator=g).tolist()
            if b not in seqs:
                seqs[b] = []
            seqs[b] = seqs[b] + ids
            lens[b], new[b] = len(seqs[b]), fed[b]
            rows += ids
            want.append(whole(m, seqs[b])[-fed[b]:])
        pad = 3
        targets = torch.randint(0, 500, (len(rows) + pad,), generator=g)
        h, lp = m.step(ints(rows + [0] * pad), ints(lens), ints(new), targets=targets.to(torch.int32).cuda(), top_k=4)
        want = torch.cat(want)
        assert dec.rel_err(h[:len(rows)].double(), want) < tol
        ref = torch.log_softmax(want @ m.head_w.double(), -1)
        got = lp.logprobs[:len(rows)].double()
        # a logit is a sum of 256 products of h; log softmax moves by at most twice the largest change
        bound = 2 * tol * want.abs().max() * m.head_w.double().abs().sum(0).max()
        assert (got - ref.gather(1, targets[:len(rows), None].cuda())[:, 0]).abs().max() < bound
        assert m.n_free.item() == 24 - sum(-(-len(s) // 8) for s in seqs.values())


def test_steps_replayed_from_one_graph(dec):
    """One captured step of 6 rows, replayed while requests grow, end and start: bit for bit the eager
    steps of a twin."""
    def make():
        return dec.T3PagedDecode(2, max_reqs=6, n_pages=30, page_size=4, max_context=40, D=128, H=2, F=256,
                                 vocab=97, seed=7)
    m, twin = make(), make()
    ids, lens, new = ints([0] * 6), ints([0] * 6), ints([0] * 6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m.step(ids, lens, new, check=False)  # warm-up on lengths of zero: nothing is allocated
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, lp = m.step(ids, lens, new, top_k=3)
    g = torch.Generator().manual_seed(8)
    n = [0] * 6
    for t in range(25):
        fed = [0] * 6
        for b in range(6):
            n[b] = 0 if (t + b) % 11 == 10 else min(n[b] + 1, 40)
            fed[b] = int(n[b] > 0 and n[b] <= 40)
        rows = torch.randint(0, 97, (6,), generator=g)
        ids.copy_(rows)
        lens.copy_(torch.tensor(n))
        new.copy_(torch.tensor(fed))
        graph.replay()
        eh, elp = twin.step(rows.to(torch.int32).cuda(), ints(n), ints(fed), top_k=3)
        live = sum(fed)
        assert torch.equal(h[:live], eh[:live]) and torch.equal(lp.top_ids[:live], elp.top_ids[:live])
        m.check_errors()
    del graph


def test_an_exhausted_pool_is_reported_and_the_next_step_runs(dec):
    m = dec.T3PagedDecode(1, max_reqs=3, n_pages=3, page_size=4, max_context=16, D=64, H=1, F=64, vocab=50)
    with pytest.raises(dec.PagedCacheFull):
        m.step(ints([1] * 18), ints([6, 6, 6]), ints([6, 6, 6]))
    with pytest.raises(dec.PagedCacheFull):  # 6 tokens are 2 pages: two requests still need 4 of the 3
        m.step(ints([1] * 12), ints([6, 0, 6]), ints([0, 0, 6]))
    m.step(ints([1] * 12), ints([4, 0, 6]), ints([0, 0, 6]))  # the first one cut back to its first page
    with pytest.raises(dec.PagedCacheFull):
        m.step(ints([1] * 3), ints([17, 0, 0]), ints([1, 0, 0]))


def test_a_length_between_the_context_and_its_last_page_is_reported(dec):
    """max_context 10 in pages of 4: lengths 11 and 12 have a page, but no position."""
    m = dec.T3PagedDecode(1, max_reqs=2, n_pages=6, page_size=4, max_context=10, D=64, H=1, F=64, vocab=50)
    m.step(ints([1] * 10), ints([10, 0]), ints([10, 0]))
    for n in (11, 12):
        with pytest.raises(dec.PagedCacheFull, match="10"):
            m.step(ints([1] * (n - 10)), ints([n, 0]), ints([n - 10, 0]))
    h, _ = m.step(ints([2, 3]), ints([10, 1]), ints([1, 1]))
    assert h.isfinite().all()


def test_a_step_without_rows_ends_requests(dec):
    m = dec.T3PagedDecode(1, max_reqs=2, n_pages=6, page_size=4, max_context=10, D=64, H=1, F=64, vocab=50)
    m.step(ints([1] * 10), ints([10, 0]), ints([10, 0]))
    h, lp = m.step(ints([]), ints([0, 0]), ints([0, 0]), top_k=2)
    assert h.shape == (0, 64) and lp.entropy.numel() == 0 and m.n_free.item() == 6
