"""PLDAGallery beside what test_gpu_grouped_callers.py holds: other streams, many tests, what is refused."""
import pytest

pytestmark = pytest.mark.gpu


def _busy():
    """Some tens of milliseconds of work on the current stream."""
    import torch

    a = torch.ones(4096, 4096, device="cuda")
    for _ in range(40):
        a = a @ a * 1e-4
    return a


def test_gallery_is_written_when_enrol_returns():
    import torch

    import synth
    from hyperion_amd.gallery import PLDAGallery
    from hyperion_amd.pdfs.plda import SPLDA

    m = synth.make_splda(40, 20)
    plda = SPLDA(mu=m["mu"], V=m["V"], W=m["W"])
    x = torch.from_numpy(synth.sample_splda(m, 30, 4, seed=5)).float().cuda()
    want = [t.clone() for t in PLDAGallery(plda).enrol(x[:100]).identify(x[100:], 4)]
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    g = PLDAGallery(plda)
    with torch.cuda.stream(one):
        keep = _busy()
        assert g.enrol(x[:100]) is g and one.query()
    with torch.cuda.stream(two):
        got = g.identify(x[100:], 4)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and keep.shape == (4096, 4096)
    assert g.gallery.k == 20 and g.rows.shape == (100,)


def _gallery(n, partitions=None, seed=3):
    """A gallery of n random vectors of a small model, and that model."""
    import numpy as np

    import synth
    from hyperion_amd.gallery import PLDAGallery
    from hyperion_amd.pdfs.plda import SPLDA

    m = synth.make_splda(24, 12)
    x = np.random.RandomState(seed).randn(n, 24).astype(np.float32)
    part = None if partitions is None else np.random.RandomState(seed + 1).randint(0, partitions, n)
    return PLDAGallery(SPLDA(mu=m["mu"], V=m["V"], W=m["W"])).enrol(x, part, partitions)


@pytest.mark.parametrize("partitions", [None, 5])
@pytest.mark.parametrize("scores", [1, 150, 1000, 4001])
def test_identify_in_slices(monkeypatch, scores, partitions):
    """However few scores fit at a time, down to those of less than one test, the answer is the same."""
    import numpy as np

    from hyperion_amd import gallery

    g = _gallery(400, partitions)
    x = np.random.RandomState(9).randn(33, 24)
    part = None if partitions is None else np.random.RandomState(8).choice([0, 1, 3], 33)
    want = g.identify(x, 6, part)
    monkeypatch.setattr(gallery, "_SLICE_BYTES", 4 * scores)
    got = g.identify(x, 6, part)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_identify_holds_few_scores_at_a_time(monkeypatch):
    """1500 tests against 400 000 rows are 2.4 GB of scores; 1 GiB of them, their mask and some more are held."""
    import numpy as np
    import torch

    from hyperion_amd import gallery

    monkeypatch.setattr(gallery, "_SLICE_BYTES", 1 << 30)
    g = _gallery(400000)
    x = torch.from_numpy(np.random.RandomState(9).randn(1500, 24)).float().cuda()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    rows, best = g.identify(x, 5)
    assert torch.cuda.max_memory_allocated() - before < 2 << 30
    at = [0, 700, 1499]
    one = [g.identify(x[i:i + 1], 5) for i in at]
    # whatever is scored together, a score is the same sum in another order of roundings at most: 64 2^-24 of its terms
    for i, (r, b) in zip(at, one):
        assert torch.equal(r[0], rows[i]) and torch.allclose(b[0], best[i], rtol=1e-5, atol=1e-4)


def test_refusals():
    import numpy as np

    import synth
    from hyperion_amd.gallery import PLDAGallery
    from hyperion_amd.pdfs.plda import SPLDA

    m = synth.make_splda(516, 513)
    with pytest.raises(ValueError, match="up to 512 latent dimensions, this one has 513"):
        PLDAGallery(SPLDA(mu=m["mu"], V=m["V"], W=m["W"]))
    g = _gallery(10)
    with pytest.raises(ValueError, match="3 partitions: say which"):
        g.enrol(np.zeros((4, 24)), num_partitions=3)
    assert g.enrol(np.ones((4, 24)), num_partitions=1).gallery.groups.num_groups == 1


def test_a_gallery_of_512_latent_dimensions():
    """A score is off by at most half a scale per coordinate times the test's projection, as for smaller models: here
    the share of its deviation that rounding to 15 levels moves, a fifth."""
    import numpy as np

    import synth
    from hyperion_amd.gallery import PLDAGallery
    from hyperion_amd.pdfs.plda import SPLDA

    m = synth.make_splda(516, 512)
    plda = SPLDA(mu=m["mu"], V=m["V"], W=m["W"])
    x = synth.sample_splda(m, 40, 6, seed=7)
    want = plda.llr_1vs1(x[::2], x[1::2])
    got = PLDAGallery(plda).enrol(x[::2]).llr(x[1::2])
    assert np.std(got - want) <= 0.2 * np.std(want)


def test_empty_galleries_and_partitions():
    import numpy as np

    g = _gallery(5)
    x = np.random.RandomState(2).randn(6, 24)
    assert g.enrol(x[:0]).llr(x).shape == (0, 6)
    rows, best = g.identify(x, 3)
    assert (rows == -1).all() and np.isneginf(best).all()
    g.enrol(x, [2, 2, 0, 2, 0, 2], 4)
    rows, best = g.identify(x, 3, [1, 3, 0, 2, 2, 1])
    assert (rows[[0, 1, 5]] == -1).all() and set(rows[2]) == {2, 4, -1} and set(rows[3]) | set(rows[4]) <= {0, 1, 3, 5}
    assert [s.shape for _, _, s in g.llr(x, [1, 3, 0, 2, 2, 1])] == [(2, 1), (0, 2), (4, 2), (0, 1)]
