"""Speculative decoding on the GPU at the edges of its arguments, against plain 64-bit implementations.

The references, the tolerances of the attention tests and their derivation are those of test_gpu_speculative.
"""
import pytest

import esolearn_b200 as E
from esolearn_b200 import _native as N
from test_gpu_speculative import IO, check_attention, gen, make_cache, ref_attention, seen_of

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
