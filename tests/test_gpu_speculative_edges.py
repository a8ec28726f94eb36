"""Speculative decoding on the GPU at the edges of its arguments, against plain 64-bit implementations.

The references, the tolerances of the attention tests and their derivation are those of test_gpu_speculative.
"""
import ctypes as C
import subprocess
import sys
import time

import pytest

import esolearn_b200 as E
from esolearn_b200 import _native as N
from test_gpu_speculative import IO, check_attention, check_verify, gen, make_cache, noise_of, parents_of, ref_attention, ref_verify, rope_tables, rows_of, seen_of, words

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    N.check(N.lib().sb_init(0))


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------
# attention

@pytest.mark.parametrize("kv,io,hd,page", [("bf16", "bf16", 128, 64), ("bf16", "f32", 64, 16), ("bf16", "bf16", 64, 7), ("int8", "f32", 128, 64)])
@pytest.mark.parametrize("ctx", [0, 5])
def test_chains_over_many_tiles_of_drafted_rows(kv, io, hd, page, ctx):
    # every tile of 128 positions holds drafted rows; a call is repeated, its result the same bit for bit
    g = gen(ctx + hd)
    t, nh, nkv = 700, 2, 1
    cache = make_cache(g, 1, ctx + t, nkv, hd, page, kv)
    q = (torch.randn(1, t, nh, hd, generator=g, device="cuda") * 2 * hd ** -0.5).to(IO[io])
    cl = ints([ctx])
    out = E.tree_attention(q, cache, cl, ctx + t)
    check_attention(out, ref_attention(q, cache, [ctx], seen_of(t)), io)
    for _ in range(50):
        assert torch.equal(out, E.tree_attention(q, cache, cl, ctx + t))


@pytest.mark.parametrize("kv", ["int8", "bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rep,t", [(1, 5), (4, 7), (3, 40), (1, 200)])
def test_a_single_seen_row_is_returned_to_f32_accuracy(kv, hd, rep, t):
    # no context, and each token sees its own row alone: the output is that row of V.  Its weight is 22 bits or more in
    # terms, each of up to six products of terms is summed in f32 with truncation (2^-23), and 1 / l, the scale and their
    # products round (2^-24 each): 4 * 2^-22 of the value in all.
    g = gen(t)
    nkv = 2
    cache = make_cache(g, 2, t, nkv, hd, 16, kv)
    q = torch.randn(2, t, rep * nkv, hd, generator=g, device="cuda") * 2 * hd ** -0.5
    mask = words(torch.eye(t, dtype=torch.bool))
    out = E.tree_attention(q, cache, ints([0, 0]), t, mask=mask)
    for b in range(2):
        want = rows_of(cache, "v", b, t).repeat_interleave(rep, 1)
        assert float(((out[b].double() - want).abs() / want.abs().clamp(min=1e-30)).max()) < 2.0 ** -20


@pytest.mark.parametrize("kv", ["int8", "bf16", "f32"])
@pytest.mark.parametrize("bad", [1e3, 1e6, -3.0e38, float("inf"), float("nan")])
@pytest.mark.parametrize("ctx", [64, 100, 127, 190])
@pytest.mark.parametrize("rep", [8])
def test_unseen_rows_beside_the_context_have_no_influence(kv, bad, ctx, rep):
    # drafted rows that share a tile with context, or begin one: what a token does not see changes no bit of its output,
    # with rep * 9 query rows per kv head
    g = gen(ctx)
    nkv, hd, t, spoilt = 2, 128, 9, 4
    cache = make_cache(g, 1, 220, nkv, hd, 16, kv)
    q = torch.randn(1, t, rep * nkv, hd, generator=g, device="cuda") * 0.1
    parents = parents_of(t, 2)
    seen = seen_of(t, parents)
    mask = torch.from_numpy(E.tree_mask(parents)).cuda()
    cl = ints([ctx])
    clean = E.tree_attention(q, cache, cl, ctx + t, mask=mask)
    check_attention(clean, ref_attention(q, cache, [ctx], seen), "f32")
    for p in [ctx + spoilt] + list(range(ctx + t, 220)):
        page, slot = int(cache.page_table[0, p // 16]), p % 16
        for x in ((cache.k_scale, cache.v_scale) if kv == "int8" else (cache.k, cache.v)):
            x[page, :, slot] = bad
    out = E.tree_attention(q, cache, cl, ctx + t, mask=mask)
    blind = ~seen[:, spoilt]
    assert 0 < int(blind.sum()) < t
    assert torch.equal(out[:, blind], clean[:, blind])


@pytest.mark.parametrize("kv", ["int8", "bf16", "f32"])
@pytest.mark.parametrize("bad", [1e3, 1e6, -3.0e38, float("inf"), float("nan")])
@pytest.mark.parametrize("ctx", [64, 100, 127, 190])
def test_unseen_rows_have_no_influence_on_few_query_rows(kv, bad, ctx):
    test_unseen_rows_beside_the_context_have_no_influence(kv, bad, ctx, 1)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("rep", [24])
@pytest.mark.parametrize("first,count", [(0, 140), (0, 3), (150, 1), (70, 60), (300, 40)])
@pytest.mark.parametrize("large", [1e3, 1e6, 1e9])
def test_seen_rows_of_large_scale_and_little_weight(io, rep, first, count, large):
    # rows of large v_scale that hardly any weight falls on, before, among and behind those that take it all, must not
    # cost these their bits (3 * rep query rows per kv head)
    g = gen(first + rep)
    nkv, hd, t, ctx = 2, 64, 3, 400
    cache = make_cache(g, 1, ctx + t, nkv, hd, 64, "int8")
    away = torch.where(torch.rand(hd, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    q = ((away + 0.1 * torch.randn(1, t, rep * nkv, hd, generator=g, device="cuda")) * 0.5).to(IO[io])
    for p in range(first, first + count):
        page, slot = int(cache.page_table[0, p // 64]), p % 64
        cache.k[page, :, slot] = (-100 * away).to(torch.int8)
        cache.k_scale[page, :, slot] = 0.03  # a score of about -96
        cache.v_scale[page, :, slot] = large
    out = E.tree_attention(q, cache, ints([ctx]), ctx + t)
    check_attention(out, ref_attention(q, cache, [ctx], seen_of(t)), io)


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("rep", [1, 4, 10])
@pytest.mark.parametrize("first,count", [(0, 1000), (0, 3), (500, 900)])
@pytest.mark.parametrize("large", [1e3, 1e6, 1e9])
def test_seen_rows_of_large_scale_that_later_scores_outweigh(io, rep, first, count, large):
    # the same with few query rows (3 to 30) and so many sequences that a warp has many tiles: rows of large v_scale that
    # it meets first, with all the weight there is so far, and that lose it to later ones
    g = gen(first + rep)
    b, nkv, hd, t, ctx = 8, 16, 64, 3, 1800
    cache = make_cache(g, b, ctx + t, nkv, hd, 64, "int8")
    away = torch.where(torch.rand(hd, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    q = ((away + 0.1 * torch.randn(b, t, rep * nkv, hd, generator=g, device="cuda")) * 0.5).to(IO[io])
    p = torch.arange(first, first + count, device="cuda")
    for i in range(b):
        page, slot = cache.page_table[i].long()[p // 64], p % 64
        cache.k[page, :, slot] = (-100 * away).to(torch.int8)
        cache.k_scale[page, :, slot] = 0.03  # a score of about -96
        cache.v_scale[page, :, slot] = large
    out = E.tree_attention(q, cache, ints([ctx] * b), ctx + t)
    check_attention(out, ref_attention(q, cache, [ctx] * b, seen_of(t)), io)


@pytest.mark.parametrize("size", [1e-10, 1e-2, 1.0])
def test_scales_of_any_size_with_many_rows(size):
    # v_scale over 12 orders of magnitude, zero scales, queries over 20, 72 query rows per kv head
    g = gen(6)
    cache = make_cache(g, 1, 400, 2, 64, 64, "int8")
    cache.v_scale.copy_(10.0 ** (torch.rand(cache.v_scale.shape, generator=g, device="cuda") * 12 - 6))
    cache.v_scale[:, :, 5] = 0
    cache.k_scale[:, :, 9] = 0
    q = torch.randn(1, 9, 16, 64, generator=g, device="cuda") * size * 0.1
    cl = ints([350])
    check_attention(E.tree_attention(q, cache, cl, 359), ref_attention(q, cache, [350], seen_of(9)), "f32")


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", ["int8", "bf16", "f32"])
@pytest.mark.parametrize("page,max_pages", [(8, 5), (7, 6), (48, 1), (16, 8), (64, 3)])
@pytest.mark.parametrize("rep", [1, 12])
def test_positions_behind_the_table_are_seen_by_no_token(kv, io, page, max_pages, rep):
    # more tokens than the table has room for (one sequence by five, one full before the call): what has no place in the
    # cache is not there, for tokens inside and outside alike, whatever shared memory held before the call
    g = gen(page + rep)
    cap, t, nkv, hd = page * max_pages, 9, 2, 64
    cache = make_cache(g, 2, cap, nkv, hd, page, kv)
    q = (torch.randn(2, t, rep * nkv, hd, generator=g, device="cuda") * 0.2).to(IO[io])
    ctx = [cap - 4, cap]
    parents = parents_of(t, 2)
    for mask, seen in ((None, seen_of(t)), (torch.from_numpy(E.tree_mask(parents)).cuda(), seen_of(t, parents))):
        out = E.tree_attention(q, cache, ints(ctx), cap + t, mask=mask)
        for b in range(2):
            k, v = (rows_of(cache, x, b, cap) for x in ("k", "v"))
            sees = torch.cat([torch.ones(t, ctx[b], dtype=torch.bool, device="cuda"), seen[:, :cap - ctx[b]]], 1)
            x = torch.einsum("tgrd,ngd->tgrn", q[b].double().view(t, nkv, rep, hd), k).masked_fill(~sees[:, None, None], -float("inf"))
            ref = torch.einsum("tgrn,ngd->tgrd", torch.softmax(x, -1), v).reshape(1, t, rep * nkv, hd)
            check_attention(out[b:b + 1], ref, io)


# ---------------------------------------------------------------------------
# the cache

@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("kv", ["int8", "bf16", "f32"])
@pytest.mark.parametrize("rope", [False, True])
def test_q_of_rows_outside_the_cache_is_zero(kv, io, rope):
    # rows on a page that does not exist, behind the table's end, before its start and behind n_new write nothing
    g = gen(2)
    cache = make_cache(g, 5, 32, 2, 64, 16, kv)
    cache.page_table[0, 1] = 10 ** 6
    cache.page_table[1, 1] = -1
    x = (torch.randn(5, 8, 8, 64, generator=g, device="cuda") + 4).to(IO[io])
    q, k, v = x.split([4, 2, 2], 2)
    q_out = torch.full((5, 8, 4, 64), 7.0, dtype=IO[io], device="cuda")
    E.kv_append(cache, k, v, ints([12, 12, 28, -3, 0]), q=q, rope=rope_tables(100, 64) if rope else None, n_new=ints([8, 8, 8, 8, 5]), q_out=q_out)
    written = [4, 4, 4, 0, 5]
    for b, n in enumerate(written):
        assert not q_out[b, n:].any() and bool(q_out[b, :n].any(-1).all())


# ---------------------------------------------------------------------------
# verification

@pytest.mark.parametrize("b,n,v,temp", [(1, 1, 8192, 1.0), (2, 1, 33000, 0.9), (64, 1, 8196, 1.0), (18, 2, 32771, 0.0), (1, 1, 400001, 0.7)])
def test_short_walks_of_several_ctas(b, n, v, temp):
    # one row a sequence, split over a cluster: the CTAs' first exchange comes soon after their start
    g = gen(b + v)
    logits = torch.randn(b, n, v, generator=g, device="cuda") * 2
    tokens = torch.zeros(b, n, dtype=torch.int32, device="cuda")
    parents = torch.arange(-1, n - 1, dtype=torch.int32, device="cuda")
    if temp == 0.0:
        best = logits.argmax(-1)
        tokens[:, 1:] = best[:, :-1].int()
        path, keep, nxt = E.verify_drafts(logits, tokens, parents, temperature=temp)
        assert keep.tolist() == [n] * b and torch.equal(nxt.long(), best[:, -1])
        return
    u = torch.rand(b, n, generator=g, device="cuda")
    noise = noise_of(g, b, v)
    first = check_verify(logits, tokens, parents, u, noise, temp)
    for _ in range(100):
        again = E.verify_drafts(logits, tokens, parents, u, noise, temperature=temp)
        assert all(torch.equal(x, y) for x, y in zip(first, again))


@pytest.mark.parametrize("b,v", [(3, 1000), (1, 1000), (4, 33001)])
@pytest.mark.parametrize("draft", [False, True])
def test_noise_shared_by_the_batch(b, v, draft):
    # one row of noise expanded over the sequences, and rows that overlap, are what their copies are
    g = gen(v)
    logits = torch.randn(b, 3, v, generator=g, device="cuda") * 2
    q = torch.softmax(logits + 0.5 * torch.randn(b, 3, v, generator=g, device="cuda"), -1) if draft else None
    tokens = logits.argmax(-1).roll(1, 1).int().contiguous()
    parents = ints([-1, 0, 1])
    u = torch.rand(b, 3, generator=g, device="cuda")
    one = noise_of(g, 1, v + 16)
    for noise in (one[:, :v].expand(b, v), one.as_strided((b, v), (4, 1))):
        got = E.verify_drafts(logits, tokens, parents, u, noise, draft_probs=q)
        want = E.verify_drafts(logits, tokens, parents, u, noise.contiguous(), draft_probs=q)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        for i in range(b):
            path, tok, near = ref_verify(logits[i], tokens[i], parents.tolist(), u[i], noise[i], 1.0, None if q is None else q[i])
            if near > 1e-4:
                assert got[0][i].tolist() == path + [-1] * (3 - len(path)) and int(got[2][i]) == tok


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("b,n,v", [(8, 5, 1000), (40, 9, 128256)])
@pytest.mark.parametrize("temp,shift", [(1e-2, 0.0), (1e-4, 0.0), (1e-6, 0.0), (0.7, 1e3), (0.7, -1e4), (0.05, 1e3)])
def test_verify_at_low_temperatures_and_shifted_logits(b, n, v, temp, shift, draft):
    """Two tokens share each row's probability and thresholds lie within 2e-4 of it, closer than a sum that is scaled
    against its terms would allow, and farther than rounding (a few 2^-24 of logits that are equal but for the gap)."""
    g = gen(n + v)
    logits = torch.randn(b, n, v, generator=g, device="cuda") * 2 + 20 * max(temp, 1.0) + shift
    top = logits.amax(-1) + 30 * temp
    pair = torch.stack([torch.randperm(v, generator=g, device="cuda")[:2] for _ in range(b * n)]).view(b, n, 2)
    # representable gaps of half a temperature or so: what the 64-bit walk sees is what the kernel is given
    logits.scatter_(2, pair, torch.stack([top, top - 0.5 * temp], -1))
    parents = torch.arange(-1, n - 1, dtype=torch.int32, device="cuda")
    p = torch.softmax(logits.double() / temp, -1)
    tokens = torch.zeros(b, n, dtype=torch.int32, device="cuda")
    tokens[:, 1:] = pair[:, :-1, 0].int()
    mine = p[:, :-1].gather(2, pair[:, :-1, :1])[..., 0]
    q = None
    if draft:  # the draft has half of that token's probability over again: accepted when u q < p
        q = torch.zeros(b, n, v, device="cuda").scatter_(2, pair, torch.stack([torch.ones(b, n, device="cuda"), torch.zeros(b, n, device="cuda")], -1))
    u = torch.rand(b, n, generator=g, device="cuda")
    near = 1 + 2e-4 * torch.where(torch.rand(b, n - 1, generator=g, device="cuda") < 0.8, -1.0, 1.0)
    u[:, 1:] = (mine * near).float()
    check_verify(logits, tokens, parents, u, noise_of(g, b, v), temp, q)


# ---------------------------------------------------------------------------
# errors of kernels

def test_a_stream_sync_costs_about_one_blocking_copy():
    # sb_stream_sync looks at the words that kernels record errors in; on an idle stream that is one small copy (a word
    # of the int8 linears), not one for each kernel
    lib = N.lib()
    word, host = torch.zeros(1, dtype=torch.int32, device="cuda"), C.c_int32()

    def best(f):
        times = []
        for _ in range(300):
            t = time.perf_counter()
            f()
            times.append(time.perf_counter() - t)
        return min(times)

    N.check(lib.sb_stream_sync(None))
    copy = best(lambda: lib.sb_memcpy_d2h(C.addressof(host), word.data_ptr(), 4, None))
    assert best(lambda: lib.sb_stream_sync(None)) < 2.5 * copy


def test_first_calls_inside_a_capture():
    # a process whose first call of an operator without a workspace is captured
    code = """
import torch, esolearn_b200 as E
cache = E.KvCache.zeros(1, 16, 1, 64, page_size=16, dtype="bf16")
cache.v.fill_(3.0)
q = torch.zeros(1, 1, 1, 64, device="cuda")
cl = torch.full((1,), 5, dtype=torch.int32, device="cuda")
out = torch.zeros_like(q)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    E.tree_attention(q, cache, cl, 6, out=out)
g.replay()
torch.cuda.synchronize()
assert bool((out == 3.0).all()), out
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


# ---------------------------------------------------------------------------
# streams and graphs

def test_first_calls_with_workspaces_inside_a_capture():
    # torch captures on a stream of its own, where no call has been made: split attention and verification both need room
    code = """
import torch, esolearn_b200 as E
cache = E.KvCache.zeros(1, 4096, 2, 128)
g = torch.Generator("cuda").manual_seed(0)
cache.k.random_(-127, 128, generator=g), cache.v.random_(-127, 128, generator=g)
cache.k_scale.fill_(0.01), cache.v_scale.fill_(0.01)
q = torch.randn(1, 4, 8, 128, generator=g, device="cuda") * 0.1
cl = torch.full((1,), 4000, dtype=torch.int32, device="cuda")
logits = torch.randn(1, 4, 32000, generator=g, device="cuda")
tokens = logits.argmax(-1).roll(1, 1).int().contiguous()
parents = torch.tensor([-1, 0, 1, 2], dtype=torch.int32, device="cuda")
u, noise = torch.rand(1, 4, generator=g, device="cuda"), torch.rand(1, 32000, generator=g, device="cuda") + 0.1
run = lambda: (E.tree_attention(q, cache, cl, 4004),) + E.verify_drafts(logits, tokens, parents, u, noise)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, run()))
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


def _step_inputs(g, b, t, v):
    x = dict(logits=torch.randn(b, t, v, generator=g, device="cuda") * 2, parents=ints(parents_of(t)), u=torch.rand(b, t, generator=g, device="cuda"),
             noise=noise_of(g, b, v), qkv=torch.randn(b, t, 8, 64, generator=g, device="cuda"))
    best = x["logits"].topk(3, -1).indices
    x["tokens"] = torch.zeros(b, t, dtype=torch.int32, device="cuda")
    for i in range(1, t):
        x["tokens"][:, i] = best[:, (i - 1) // 3, (i - 1) % 3].int()
    return x


def _step(x, cache, cl):
    """Append, attention, verification, commit and read of one step."""
    q, k, v = x["qkv"].split([4, 2, 2], 2)
    q = E.kv_append(cache, k, v, cl, q=q, rope=x["rope"], q_scale=0.125)
    y = E.tree_attention(q, cache, cl, 400, mask=x["mask"])
    path, keep, nxt = E.verify_drafts(x["logits"], x["tokens"], x["parents"], x["u"], x["noise"], temperature=0.9)
    E.kv_commit(cache, cl, path, keep)
    return (y, path, keep, nxt) + E.kv_read(cache, 20, start=cl)


def _step_setup(seed, b, t, v):
    g = gen(seed)
    x = _step_inputs(g, b, t, v)
    x["rope"] = rope_tables(400, 64)
    x["mask"] = torch.from_numpy(E.tree_mask(parents_of(t))).cuda()
    return x, make_cache(g, b, 400, 2, 64, 16, "int8"), ints([300 - 20 * i for i in range(b)])


@pytest.mark.parametrize("b,t,v", [(2, 13, 5000), (3, 13, 128256), (12, 20, 33001)])
def test_a_step_on_several_streams(b, t, v):
    """Steps of different sequences on two streams at once are what they are one after the other."""
    steps = [_step_setup(s, b, t, v) for s in range(2)]
    start = [[c.k.clone(), c.v.clone(), c.k_scale.clone(), c.v_scale.clone()] for _, c, _ in steps]
    want = [_step(*s) for s in steps]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for (x, c, cl), old in zip(steps, start):
            for dst, src in zip((c.k, c.v, c.k_scale, c.v_scale), old):
                dst.copy_(src)
        torch.cuda.synchronize()
        got = []
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                got.append(_step(*s))
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, c))


@pytest.mark.parametrize("b,t,v", [(2, 13, 5000), (3, 13, 128256), (12, 20, 33001)])
def test_a_step_in_a_graph(b, t, v):
    """A captured step, replayed on new inputs in the same tensors, is the step called directly."""
    x, cache, cl = _step_setup(5, b, t, v)
    parts = (cache.k, cache.v, cache.k_scale, cache.v_scale)
    old = [p.clone() for p in parts]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _step(x, cache, cl)  # its workspaces
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = _step(x, cache, cl)
    for seed in (6, 7):
        new = _step_inputs(gen(seed), b, t, v)
        for name in new:
            x[name].copy_(new[name])
        for p, o in zip(parts, old):
            p.copy_(o)
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in out] + [p.clone() for p in parts]
        for p, o in zip(parts, old):
            p.copy_(o)
        want = list(_step(x, cache, cl)) + list(parts)
        assert all(torch.equal(a, c) for a, c in zip(got, want))
