"""sample_logits where rows are cut into slices of several lengths."""
import numpy as np
import pytest

from sample_cases import Sample, distribution

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [8193, 16384, 40000, 60000, 70001])
@pytest.mark.parametrize("far", [31.5, 32.0, 32.5])
def test_weights_next_to_nothing_count_alike_in_every_slice(gpu, vocab, far):
    """All tokens but the last weigh about 2^-46 of it, and numbers fall among
    them or past them: a row is drawn alike among few rows and among many, whose
    slices are longer, and through the scratch."""
    row = np.full((1, vocab), -far, np.float32)
    row[0, vocab - 1] = 0
    u = (2.0 ** -np.arange(28, 48)).astype(np.float32)
    few = Sample(row.repeat(len(u), axis=0), u=u)
    tokens, probs = few.run(gpu)
    many = Sample(row.repeat(15 * len(u), axis=0), u=np.tile(u, 15))
    for static in (False, True):
        got, shares = many.run(gpu, static=static)
        assert (got.reshape(15, -1) == tokens).all() and (shares.reshape(15, -1) == probs).all()
    for i in range(0, len(u), 7):
        got, share = Sample(row, u=u[i:i + 1]).run(gpu)
        assert got[0] == tokens[i] and share[0] == probs[i]


@pytest.mark.parametrize("vocab", [5000, 20000])
@pytest.mark.parametrize("temperature", [1e12, 1e15, 1e18, 1e30, np.inf])
@pytest.mark.parametrize("min_p", [0.5, np.nextafter(np.float32(1), np.float32(0)), 1.0])
def test_temperatures_far_above_the_logits(gpu, vocab, temperature, min_p):
    """Weights all but equal, of which min_p keeps those that reach it in 64 bits."""
    rng = np.random.default_rng(vocab)
    case = Sample(3 * rng.standard_normal((6, vocab)), temperature, min_p=min_p, u=[0, 1, 0.25, *rng.random(3)])
    tokens, _ = case.check(gpu)
    if temperature == 1e18:
        assert len(distribution(case.logits[0], 1e18, 0, 1.0, min_p)[0]) == vocab and tokens[0] == 0
