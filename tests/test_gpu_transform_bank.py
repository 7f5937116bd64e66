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


def _busy():
    """Some tens of milliseconds of work on the current stream."""
    import torch

    a = torch.ones(4096, 4096, device="cuda")
    for _ in range(40):
        a = a @ a * 1e-4
    return a


def test_maps_are_written_when_their_constructor_returns():
    import torch

    from hyperion_amd import engine

    rng = np.random.RandomState(1)
    W, x = torch.from_numpy(rng.randn(2, 30, 20)).float().cuda(), torch.from_numpy(rng.randn(50, 30)).float().cuda()
    groups = engine.RowGroups([20, 30])
    want = engine.grouped_affine(x, groups, engine.AffineBank(W))
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(one):
        keep = _busy()
        bank = engine.AffineBank(W)
        assert one.query()
    with torch.cuda.stream(two):
        got = engine.grouped_affine(x, groups, bank)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and keep.shape == (4096, 4096)
    graph = torch.cuda.CUDAGraph()  # made inside a capture they are part of it
    with torch.cuda.graph(graph):
        inside = engine.grouped_affine(x, groups, engine.AffineBank(W))
    for scale in (1, 2):
        W.mul_(scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(inside, want * scale)


def test_predict_on_a_second_stream_right_after_the_first():
    """The maps that the first call on one stream lays out are there for a call on another that waits for nothing."""
    import torch

    from hyperion_amd import engine
    from hyperion_amd.transforms import CentWhiten, LNorm, TransformBank

    rng = np.random.RandomState(2)
    d, n = 64, 300
    chains = [[CentWhiten(mu=rng.randn(d), T=rng.randn(d, d)), LNorm()] for _ in range(3)]
    groups = engine.RowGroups([100, 150, 50])
    x = torch.from_numpy(rng.randn(n, d)).float().cuda()
    want = TransformBank(chains).predict(x, groups)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        bank = TransformBank(chains)
        with torch.cuda.stream(one):
            keep = _busy()
            first = bank.predict(x, groups)
        with torch.cuda.stream(two):
            second = bank.predict(x, groups)
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(second, want) and keep.shape == (4096, 4096)


def test_predict_from_two_threads_at_once():
    """Two threads, each on a stream of its own, whose vectors have different dimensions and so need different maps."""
    import threading

    import torch

    from hyperion_amd import engine
    from hyperion_amd.transforms import LNorm, TransformBank

    rng = np.random.RandomState(3)
    bank = TransformBank([[LNorm(), LNorm()], [LNorm(), LNorm()]])
    groups = engine.RowGroups([40, 60])
    xs = [torch.from_numpy(rng.randn(100, d)).float().cuda() for d in (16, 40)]
    wants = [TransformBank(bank.chains).predict(x, groups) for x in xs]
    torch.cuda.synchronize()
    errors = []

    def work(x, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    got = bank.predict(x, groups)
                    torch.cuda.current_stream().synchronize()
                    if not torch.equal(got, want):
                        errors.append("differs")
        except Exception as e:  # an error of either thread fails the test
            errors.append(e)

    threads = [threading.Thread(target=work, args=a) for a in zip(xs, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
