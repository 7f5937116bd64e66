"""TransformBank: maps laid out for one set of chains are not used for another, nor before they are written."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_maps_follow_a_change_of_the_chains():
    """A step that moves to another chain and a centring that becomes a length normalisation keep all parameters and
    their order; what is computed changes.  The bar is that of the parity tests, 1e-4 max(|y|, 1)."""
    from hyperion_amd.transforms import CentWhiten, LNorm, TransformBank, TransformList

    rng = np.random.RandomState(0)
    n, d = 40, 24
    x, ids = rng.randn(n, d) + 2, np.arange(n) % 2
    L, A = LNorm(), CentWhiten(mu=rng.randn(d), T=rng.randn(d, d) / np.sqrt(d))
    bank = TransformBank([[L], [A, L]])

    def check():
        y = bank.predict(x, ids)
        for e, chain in enumerate(bank.chains):
            want = TransformList(list(chain)).predict(x[ids == e])
            assert (np.abs(y[ids == e] - want) <= 1e-4 * np.maximum(np.abs(want), 1)).all()

    check()
    bank.chains = [[L, A], [L]]
    check()
    bank.chains = [[CentWhiten(), A], [CentWhiten()]]
    check()
    bank.chains = [[LNorm(), A], [LNorm()]]
    check()
    single = TransformList([CentWhiten(mu=A.mu, T=A.T)])
    before = single.predict(x)
    single.transforms[0] = LNorm(mu=A.mu, T=A.T)
    after = single.predict(x)
    want = before * np.sqrt(d) / np.linalg.norm(before, axis=1, keepdims=True)
    assert (np.abs(after - want) <= 1e-4 * np.maximum(np.abs(want), 1)).all()
