"""Speculative decoding on the GPU at the edges of its arguments, against plain 64-bit implementations.

The references, the tolerances of the attention tests and their derivation are those of test_gpu_speculative.
"""
import pytest

import esolearn_b200 as E
from esolearn_b200 import _native as N
from test_gpu_speculative import IO, check_attention, check_verify, gen, make_cache, noise_of, ref_attention, ref_verify, seen_of

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
