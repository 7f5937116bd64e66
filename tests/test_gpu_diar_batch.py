"""DiarAHCPLDA.scores_batch / cluster_batch beside what test_gpu_grouped_callers.py holds."""
import numpy as np
import pytest

import synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("y_dim", [510, 511, 512])
@pytest.mark.parametrize("var_r", [1, 0.85])
def test_models_of_many_latent_dimensions(var_r, y_dim):
    """Packed rows of 512 (510 dimensions) are the widest of the grouped product; wider ones are scored one recording
    at a time.  Projected rows are off by less than 2^-17 in fp32, of terms of some ten times the largest score: 1e-4 of
    it."""
    from hyperion_amd.diarization import DiarAHCPLDA
    from hyperion_amd.pdfs.plda import SPLDA

    m = synth.make_splda(520, y_dim)
    diar = DiarAHCPLDA(SPLDA(mu=m["mu"], V=m["V"], W=m["W"]), threshold=0.0, pca_var_r=var_r)
    x = synth.sample_splda(m, 12, 9, seed=3)
    xs = [x[:40], x[40:43], x[43:]]
    got = diar.scores_batch(xs)
    for a, x in zip(got, xs):
        want = diar.scores(x).cpu().numpy()
        assert a.shape == want.shape
        assert np.abs(a.cpu().numpy() - want).max() <= 1e-4 * np.abs(want).max()
    for ids, x in zip(diar.cluster_batch(xs + [x[:1]]), xs):
        assert np.array_equal(ids, diar.cluster(x))
