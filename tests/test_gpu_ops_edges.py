"""The token-step operators at the values and uses where they can go wrong: infinities beside masked places, exact products, eps 0, tensors that
carry gradients, several callers of one handle.  Plain implementations and bounds as in test_gpu_ops.py."""
import math

import pytest
import torch

from test_gpu_ops import ACT, Paged, ints, ops, rnd  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------------------------
# attention
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv,rep", [(1, 1), (2, 2), (1, 4), (2, 7)])
@pytest.mark.parametrize("lens,window", [([21, 32, 1, 129], 0), ([33, 70, 500, 31], 27), ([3000, 45, 1, 1027], 0), ([3000, 2011], 1999)])
def test_attention_of_an_infinity_in_a_32_bit_cache(ops, hd, kv, rep, lens, window):  # noqa: F811
    """A 32-bit cache keeps its values: an infinity that is seen is the result of its column, and no other column, head or sequence changes.  It
    stands in the last token, the first that is seen, and one between; the places behind and before are masked."""
    P = Paged(ops, lens, kv, hd, 16, "f32", seed=hd + rep)
    q = rnd((len(lens), kv * rep, hd), torch.float32, 5).cuda()
    want, lse = ops.attention(q, P.cache, P.table, P.lens_dev, window=window, lse=True)
    ops.sync()
    assert bool(want.isfinite().all())
    for b, n in enumerate(lens):
        low = max(0, n - window) if window else 0
        for i, t in enumerate({n - 1, low, (low + n) // 2}):
            page, head, col = int(P.table[b, t // 16]), (i + 1) % kv, (7 * i + 3) % hd
            kept = float(P.cache.v[page, head, t % 16, col])
            P.cache.v[page, head, t % 16, col] = -math.inf if i == 1 else math.inf
            out, got = ops.attention(q, P.cache, P.table, P.lens_dev, window=window, lse=True)
            ops.sync()
            P.cache.v[page, head, t % 16, col] = kept
            expect = want.clone()
            expect[b, head * rep:(head + 1) * rep, col] = -math.inf if i == 1 else math.inf
            assert torch.equal(out, expect) and torch.equal(got, lse), (b, t)
