"""Refusals of the paged entry points and cbx_token_logprobs, and their plain
definitions: no GPU needed (every refused call returns before any CUDA call)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from _paged import attention_ref, logprobs_ref, plan_ref


@pytest.fixture(scope="module")
def lib():
    import os

    from chatterbox_amdvulkan_b200 import _lib, build
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    return _lib.load()


def P(i):
    """A made-up device address, never dereferenced: every call below fails before a launch."""
    return ctypes.c_void_p(0x100000 * i)


def plan_args(**kw):
    a = dict(lens=P(1), new=None, B=4, mb=8, page=16, pages=32, ti=P(2), bi=P(3), fi=P(4), ni=P(5),
             to=P(6), bo=P(7), fo=P(8), no=P(9), rows=4, slots=P(10), pos=P(11), reqs=None, rl=None,
             start=None, err=P(12), stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(B=-1), "n_reqs"), (dict(B=8193), "n_reqs"), (dict(mb=0), "max_blocks"),
    (dict(B=8192, mb=1 << 20), "max_blocks"), (dict(page=0), "page_size"), (dict(pages=0), "n_pages"),
    (dict(page=1 << 20, pages=1 << 12), "n_pages"), (dict(rows=-1), "max_rows"),
    (dict(rows=1 << 31), "max_rows"), (dict(lens=None), "NULL"), (dict(to=None), "NULL"),
    (dict(err=None), "NULL"), (dict(slots=None), "NULL"), (dict(fo=None), "NULL"),
    (dict(to=P(3)), "overlaps an input"), (dict(fo=P(2)), "overlaps an input"),
    (dict(slots=P(1)), "overlaps an input"), (dict(pos=P(10)), "outputs overlap"),
    (dict(to=ctypes.c_void_p(0x200004)), "overlaps an input"),       # shifted by one entry
    (dict(reqs=P(6)), "outputs overlap"), (dict(start=P(7)), "outputs overlap"),
])
def test_plan_refusals(lib, kw, msg):
    assert lib.cbx_paged_plan(*plan_args(**kw)) == -1
    assert msg in lib.cbx_last_error().decode()


def append_args(**kw):
    a = dict(qkv=P(1), t=0, stride=0, bias=None, n=2, qd=64, kd=32, slots=P(2), ck=P(3), cv=P(4), ct=0,
             pages=4, page=16, ps=0, q=None, err=P(5), stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,status,msg", [
    (dict(n=-1), -1, "n_rows"), (dict(kd=0), -1, "kv_dim"), (dict(qd=-8), -1, "q_dim"),
    (dict(stride=127), -1, "qkv_row_stride"), (dict(page=0), -1, "page_size"),
    (dict(pages=0), -1, "n_pages"), (dict(pages=1 << 28, page=16), -1, "n_pages"),
    (dict(ps=16 * 32 - 1), -1, "pages overlap"), (dict(t=9), -2, "qkv_type"),
    (dict(ct=9), -2, "cache_type"), (dict(qkv=None), -1, "NULL"), (dict(slots=None), -1, "NULL"),
    (dict(cv=None), -1, "NULL"), (dict(err=None), -1, "NULL"),
])
def test_append_refusals(lib, kw, status, msg):
    assert lib.cbx_qkv_kv_append_paged(*append_args(**kw)) == status
    assert msg in lib.cbx_last_error().decode()
    assert lib.cbx_qkv_kv_append_paged(*append_args(n=0, qkv=None)) == 0


def attn_args(**kw):
    a = dict(q=P(1), qt=0, qs=0, ck=P(2), cv=P(3), ct=0, pages=64, page=16, ps=0, table=P(4), reqs=2,
             mb=8, rr=None, lens=P(5), rows=2, H=4, Hk=2, hd=64, scale=0.125, out=P(6), lse=None,
             ws=None, wsb=0, err=P(7), stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,status,msg", [
    (dict(rows=-1), -1, "n_rows"), (dict(rows=1 << 31), -1, "n_rows"), (dict(rows=1 << 29, reqs=1 << 29), -1, "2^31"), (dict(H=5), -1, "multiple"),
    (dict(Hk=0), -1, "multiple"), (dict(hd=60), -1, "head_dim"), (dict(hd=264), -1, "head_dim"),
    (dict(hd=0), -1, "head_dim"), (dict(mb=0), -1, "max_blocks"), (dict(page=0), -1, "page_size"),
    (dict(pages=0), -1, "n_pages"), (dict(ps=16 * 128 - 128), -1, "page_stride"),
    (dict(ps=16 * 128 + 8), -1, "page_stride"), (dict(pages=1 << 26, ps=64 * 128), -1, "rows"),
    (dict(qs=255), -1, "q_row_stride"), (dict(reqs=1), -1, "n_reqs"), (dict(qt=5), -2, "q_type"),
    (dict(ct=5), -2, "cache_type"), (dict(q=None), -1, "NULL"), (dict(out=None), -1, "NULL"),
    (dict(err=None), -1, "NULL"), (dict(ck=ctypes.c_void_p(0x200008)), -1, "aligned"),
])
def test_attention_refusals(lib, kw, status, msg):
    assert lib.cbx_paged_decode_attention(*attn_args(**kw)) == status
    assert msg in lib.cbx_last_error().decode()


def test_attention_workspace(lib):
    ws = lib.cbx_paged_decode_attention_workspace
    assert ws(0, 16, 16, 64, 128, 16, 0) == 0
    assert ws(4, 16, 3, 64, 128, 16, 0) == -1 and "multiple" in lib.cbx_last_error().decode()
    assert ws(4, 16, 4, 64, 128, 16, 7) == -2
    assert ws(65535, 64, 8, 128, 8, 16, 30) == 0          # enough rows: no split over the keys
    need = ws(1, 1, 1, 128, 65536, 16, 30)                # one row of one head over 2^20 keys
    assert need > 0
    big = dict(rows=1, H=1, Hk=1, hd=128, mb=65536, reqs=1, ct=30)
    assert lib.cbx_paged_decode_attention(*attn_args(**big)) == -1
    assert "workspace" in lib.cbx_last_error().decode()
    assert lib.cbx_paged_decode_attention(*attn_args(**big, ws=P(9), wsb=need - 1)) == -1
    assert lib.cbx_paged_decode_attention(*attn_args(**big, ws=ctypes.c_void_p(0x900004), wsb=need)) == -1


@pytest.mark.parametrize("args,status,msg", [
    ((P(1), 0, 0, -1, 8, None, 0, None, None, None, None, None, None), -1, "n_rows"),
    ((P(1), 0, 0, 2, 0, None, 0, None, None, None, None, None, None), -1, "vocab"),
    ((P(1), 0, 7, 2, 8, None, 0, None, None, None, None, None, None), -1, "row_stride"),
    ((P(1), 4, 0, 2, 8, None, 0, None, None, None, None, None, None), -2, "type"),
    ((P(1), 0, 0, 2, 8, None, 9, None, None, P(2), P(3), None, None), -1, "top_k"),
    ((P(1), 0, 0, 2, 80, None, 33, None, None, P(2), P(3), None, None), -1, "top_k"),
    ((P(1), 0, 0, 2, 80, None, -1, None, None, P(2), P(3), None, None), -1, "top_k"),
    ((None, 0, 0, 2, 8, None, 0, None, P(2), None, None, None, None), -1, "NULL"),
    ((P(1), 0, 0, 2, 8, P(2), 0, None, None, None, None, P(3), None), -1, "NULL"),
    ((P(1), 0, 0, 2, 8, P(2), 0, P(3), None, None, None, None, None), -1, "NULL"),
    ((P(1), 0, 0, 2, 8, None, 2, None, None, P(2), None, None, None), -1, "NULL"),
    ((ctypes.c_void_p(0x100002), 0, 0, 2, 8, None, 0, None, P(2), None, None, None, None), -1, "aligned"),
])
def test_logprobs_refusals(lib, args, status, msg):
    assert lib.cbx_token_logprobs(*args) == status
    assert msg in lib.cbx_last_error().decode()
    assert lib.cbx_token_logprobs(None, 0, 0, 0, 8, None, 0, None, None, None, None, None, None) == 0


def test_wrappers_refuse_before_the_device(lib):
    """The torch wrappers know the tensors' shapes: they refuse them before anything is launched,
    and CPU tensors after that."""
    from chatterbox_amdvulkan_b200 import ops
    i32 = torch.int32
    z = lambda *s: torch.zeros(*s, dtype=i32)  # noqa: E731
    plan = dict(seq_lens=z(3), block_table=z(3, 4), n_blocks=z(3), free_list=z(20), n_free=z(1), page_size=16)
    for bad, msg in ((dict(block_table=z(2, 4)), "block_table"), (dict(n_blocks=z(2)), "n_blocks"),
                     (dict(n_new=z(4)), "n_new"), (dict(out=[z(3)] * 9), "out must"),
                     (dict(out=[z(3)] * 9, in_place=True), "exclude"), ({}, "CUDA")):
        with pytest.raises(ValueError, match=msg):
            ops.paged_plan(**{**plan, **bad})
    k = torch.zeros(5, 16, 2, 32)
    app = dict(qkv=torch.zeros(3, 4 * 32 + 2 * 64), bias=None, cache_k=k, cache_v=k.clone(), slots=z(3))
    for bad, msg in ((dict(qkv=torch.zeros(3, 100)), "below"), (dict(slots=z(2)), "slots"),
                     (dict(bias=torch.zeros(7)), "bias"), (dict(cache_v=k[:4]), "one shape"),
                     (dict(cache_k=k[:, ::2], cache_v=k[:, ::2]), "dense"),
                     (dict(cache_v=torch.zeros(10, 16, 2, 32)[::2]), "equally"),
                     (dict(q_out=torch.zeros(3, 4)), "q_out"), (dict(qkv=torch.zeros(256, 3).T), "dense"), ({}, "CUDA")):
        with pytest.raises(ValueError, match=msg):
            ops.qkv_kv_append_paged(**{**app, **bad})
    with pytest.raises(TypeError, match="dtype"):
        ops.qkv_kv_append_paged(**{**app, "cache_v": k.half()})
    at = dict(q=torch.zeros(3, 4, 32), cache_k=k, cache_v=k.clone(), block_table=z(3, 4), seq_lens=z(3))
    for bad, msg in ((dict(q=torch.zeros(3, 4, 64)), "head_dim"), (dict(seq_lens=z(2)), "seq_lens"),
                     (dict(block_table=z(2, 4)), "block_table"), (dict(row_reqs=z(4)), "row_reqs"),
                     (dict(out=torch.zeros(3, 4, 31)), "out"), (dict(q=torch.zeros(3, 32, 4).transpose(1, 2)), "dense"),
                     (dict(q=torch.zeros(1, 4, 32).expand(3, 4, 32)), "overlap"), ({}, "CUDA")):
        with pytest.raises(ValueError, match=msg):
            ops.paged_decode_attention(**{**at, **bad})
    x = torch.zeros(3, 40)
    for kw, msg in ((dict(logits=x, tokens=z(2)), "tokens"), (dict(logits=x, tokens=None, top_k=33), "top_k"),
                    (dict(logits=x[:, :4], tokens=None, top_k=5), "top_k"), (dict(logits=x.T, tokens=None), "dense"),
                    (dict(logits=x[:1].expand(3, 40), tokens=None), "overlap"), (dict(logits=x, tokens=z(3)), "CUDA")):
        with pytest.raises(ValueError, match=msg):
            ops.token_logprobs(**kw)


def test_plan_definition_on_an_example():
    """Two pages of 4 tokens come back from a request that ended, one is popped again."""
    s, p, r, n, start, table, have, free, n_free, flags = plan_ref(
        [0, 5, 3], [0, 1, 3], [[7, 2], [1, -1], [-1, -1]], [2, 1, 0], [5, 0, 0, 0, 0, 0, 0, 0], 1, 4, 5)
    assert (table, have, flags) == ([[-1, -1], [1, 2], [7, -1]], [0, 2, 1], 0)
    assert (s, p, r, n) == ([8, 28, 29, 30, -1], [4, 0, 1, 2, 0], [1, 2, 2, 2, 0], [5, 1, 2, 3, 0])
    assert (start, n_free, free[:1]) == ([0, 0, 1, 4], 1, [5])


def test_definitions_agree_with_torch():
    """The 64-bit definitions against torch's own attention and log_softmax."""
    g = torch.Generator().manual_seed(1)
    ck, cv = (torch.randn(6, 4, 2, 8, generator=g, dtype=torch.float64) for _ in range(2))
    q = torch.randn(2, 4, 8, generator=g, dtype=torch.float64)
    table = torch.tensor([[3, 1, 5], [0, 2, -1]], dtype=torch.int32)
    out, lse, _ = attention_ref(q, ck, cv, table, torch.tensor([11, 0]))
    k = ck[[3, 1, 5]].flatten(0, 1)[:11].repeat_interleave(2, 1).transpose(0, 1)
    v = cv[[3, 1, 5]].flatten(0, 1)[:11].repeat_interleave(2, 1).transpose(0, 1)
    ref = torch.nn.functional.scaled_dot_product_attention(q[0][:, None], k, v)[:, 0]
    assert torch.allclose(out[0], ref, atol=1e-12) and not out[1].any() and (lse[1] == -torch.inf).all()
    x = torch.randn(3, 50, generator=g, dtype=torch.float64)
    lp, ent, ids, top, _, _ = logprobs_ref(x, torch.tensor([1, 2, 3]), 4)
    y = torch.log_softmax(x, -1)
    assert torch.allclose(lp, y[[0, 1, 2], [1, 2, 3]]) and torch.allclose(ent, torch.distributions.Categorical(logits=x).entropy())
    assert torch.allclose(top, y.topk(4).values)


class OnDevice1(torch.Tensor):
    """A host tensor that says it is on CUDA device 1."""
    def get_device(self):
        return 1


def test_wrappers_run_with_their_tensors_device_current(monkeypatch):
    """Tensors on device 1 while device 0 is current, the arguments in any order of keywords: every call
    reaches the library with device 1 current, or is refused."""
    from chatterbox_amdvulkan_b200 import ops
    state, calls = {"dev": 0}, []

    class Device:
        def __init__(self, dev):
            self.dev = dev

        def __enter__(self):
            self.before, state["dev"] = state["dev"], self.dev

        def __exit__(self, *a):
            state["dev"] = self.before

    monkeypatch.setattr(ops, "_current_device", lambda: state["dev"])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: None)
    monkeypatch.setattr(ops, "_workspace_bytes", lambda *a: 0)
    monkeypatch.setattr(ops, "_fn", lambda name: lambda *a: calls.append((name, state["dev"])) or 0)

    def on1(t):
        return t.as_subclass(OnDevice1)

    def z(*s):
        return on1(torch.zeros(*s, dtype=torch.int32))

    k = on1(torch.zeros(5, 16, 2, 32))
    err = z(1)
    plan = dict(page_size=16, err=err, n_new=None, max_rows=3, free_list=z(20), n_free=z(1), block_table=z(3, 4),
                n_blocks=z(3), out=[z(n) for n in (3, 3, 3, 3, 4, 12, 3, 20, 1)], seq_lens=z(3))
    append = dict(bias=None, with_q=True, err=err, slots=z(3), cache_k=k, cache_v=k, qkv=on1(torch.zeros(3, 256)))
    attend = dict(scale=1.0, row_reqs=None, err=err, seq_lens=z(3), block_table=z(3, 4), cache_k=k, cache_v=k,
                  q=on1(torch.zeros(3, 4, 32)))
    score = dict(top_k=2, tokens=None, err=err, logits=on1(torch.zeros(3, 40)))
    for fn, kw in ((ops.paged_plan, plan), (ops.qkv_kv_append_paged, append), (ops.paged_decode_attention, attend),
                   (ops.token_logprobs, score)):
        fn(**kw)
        fn(**dict(reversed(kw.items())))
        first, *rest = reversed(kw.items())
        fn(first[1], **dict(rest))
    assert len(calls) == 12 and all(dev == 1 for _, dev in calls) and state["dev"] == 0
    # one tensor on the host, or on another device, is refused
    other = torch.zeros(3, dtype=torch.int32)
    for fn, kw in ((ops.paged_plan, {**plan, "n_blocks": other}), (ops.qkv_kv_append_paged, {**append, "slots": other}),
                   (ops.paged_decode_attention, {**attend, "seq_lens": other}),
                   (ops.token_logprobs, {**score, "tokens": other})):
        with pytest.raises(ValueError):
            fn(**kw)
    assert len(calls) == 12


def at(addr):
    return ctypes.c_void_p(addr)


def test_misaligned_arguments_are_refused(lib):
    """Every pointer of the paged entry points and of cbx_token_logprobs, two bytes (one for 16-bit data) off
    its type's boundary: refused before a launch."""
    for name in ("lens", "new", "ti", "bi", "fi", "ni", "to", "bo", "fo", "no", "slots", "pos", "reqs", "rl", "start", "err"):
        assert lib.cbx_paged_plan(*plan_args(**{name: at(0x2000002)})) == -1
        assert "aligned" in lib.cbx_last_error().decode(), name
    for name, t, ct, off in (("qkv", 0, 0, 2), ("qkv", 1, 0, 1), ("q", 0, 0, 2), ("q", 1, 0, 1), ("ck", 0, 0, 2),
                             ("cv", 0, 1, 1), ("bias", 0, 0, 2), ("slots", 0, 0, 2), ("err", 0, 0, 2)):
        assert lib.cbx_qkv_kv_append_paged(*append_args(**{name: at(0x2000000 + off), "t": t, "ct": ct})) == -1
        assert "aligned" in lib.cbx_last_error().decode(), name
    for name, qt, off in (("q", 0, 2), ("q", 1, 1), ("out", 0, 2), ("out", 1, 1), ("table", 0, 2), ("rr", 0, 2),
                          ("lens", 0, 2), ("lse", 0, 2), ("err", 0, 2)):
        assert lib.cbx_paged_decode_attention(*attn_args(**{name: at(0x2000000 + off), "qt": qt})) == -1
        assert "aligned" in lib.cbx_last_error().decode(), name
    good = [P(1), 0, 0, 2, 80, P(2), 4, P(3), P(4), P(5), P(6), P(7), None]
    for i in (0, 5, 7, 8, 9, 10, 11):
        assert lib.cbx_token_logprobs(*good[:i], at(0x2000002), *good[i + 1:]) == -1
        assert "aligned" in lib.cbx_last_error().decode(), i


def test_outputs_over_their_inputs_are_refused(lib):
    """Heads and rows are worked on side by side: attention cannot write over q, nor the epilogue its q over
    qkv.  Two rows of 4 x 64 f32 at 0x100000; a row of gap behind each is free."""
    row = 4 * 64 * 4
    for off in (0, 4, row, 2 * row - 4, 4 - 2 * row):
        assert lib.cbx_paged_decode_attention(*attn_args(out=at(0x100000 + off))) == -1
        assert "overlaps q" in lib.cbx_last_error().decode(), off
    assert lib.cbx_paged_decode_attention(*attn_args(lse=at(0x100000 + 64))) == -1
    assert "overlaps q" in lib.cbx_last_error().decode()
    wide = dict(qs=4 * 256)  # rows four rows apart
    for off in (4 - 2 * row, 0, 3 * row - 4, 2 * row + 4, 4 * row, 5 * row - 4):
        assert lib.cbx_paged_decode_attention(*attn_args(out=at(0x100000 + off), **wide)) == -1
        assert "overlaps q" in lib.cbx_last_error().decode(), off
    # where they do not meet, the next check answers (the caches' alignment)
    for off in (-2 * row, row, 2 * row, 5 * row):
        assert lib.cbx_paged_decode_attention(*attn_args(out=at(0x100000 + off), ck=at(0x200008), **wide)) == -1
        assert "16-byte" in lib.cbx_last_error().decode(), off
    for off in (0, 512, 2 * 512 - 4, 4 - 2 * 64 * 4):  # two rows of 128 f32, q of 64
        assert lib.cbx_qkv_kv_append_paged(*append_args(q=at(0x100000 + off))) == -1
        assert "overlaps qkv" in lib.cbx_last_error().decode(), off
