"""The sums behind log probabilities and entropies of long rows in one block each: small
terms behind large ones are not lost."""
import numpy as np
import pytest

import int8_reference as ref

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,low", [(torch.bfloat16, -13.25), (torch.float32, -14.0)])
def test_small_terms_behind_large_ones(dtype, low):
    """The first tile's logits are 0, all others so low that each term is below half a step of the 32
    (F32: 16) that a thread's sum holds by then, while together they are 5e-5 of it.

    Each s is a sum of at most 32 terms of a tile, of 61 tiles at most, 6 steps of a wave's
    lanes and 2 of the waves: with the terms' own errors (two steps, and 2.5 u |x - m|, whose weighted
    mean is below 1 here) off by at most (31 + 61 + 8 + 2 + 3) u. log s rounds within two steps;
    the entropy adds the same for t (in terms of the weighted mean, below 0.01) and two roundings."""
    print("small terms", dtype, flush=True)
    import cq35
    rows, vocab = 520, 248320  # too many rows for several blocks each
    tile = 16 // dtype.itemsize * 4 * 256
    x = torch.full((1, vocab), low, dtype=dtype, device="cuda")
    x[0, :tile] = 0.0
    t = torch.tensor([[0, vocab - 1]], device="cuda")
    got = cq35.token_logprobs(x.expand(rows, vocab), t.repeat(rows, 1), top=1)
    lp, entropy, best, _ = ref.logprobs(x, t, 1)
    log_s = -lp[0, 0]
    limit = 105 * ref.U + 4 * ref.U * log_s
    assert np.abs(got.logprobs[:, 0].cpu().double().numpy() - lp[0, 0]).max() <= limit
    assert np.abs(got.logprobs[:, 1].cpu().double().numpy() - lp[0, 1]).max() <= limit + 2 * ref.U * abs(lp[0, 1])
    assert np.abs(got.entropy.cpu().double().numpy() - entropy[0]).max() <= limit + 0.01 * 2 * 105 * ref.U + 2 * ref.U * entropy[0]
    assert bool((got.top_tokens == 0).all())


def test_results_of_another_number_are_refused():
    print("results", flush=True)
    import cq35
    x, t = torch.zeros(3, 50, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    whole = cq35.token_logprobs(x, t, top=2)
    for out in (whole[:3], whole[:2], (), list(whole) + [whole[0]], x, 5):
        with pytest.raises(TypeError, match="four tensors"):
            cq35.token_logprobs(x, t, top=2, out=out)
    assert cq35.token_logprobs(x, t, top=2, out=list(whole)).entropy is whole.entropy
