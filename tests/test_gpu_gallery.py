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
