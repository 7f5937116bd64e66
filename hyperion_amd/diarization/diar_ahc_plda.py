import numpy as np

from .. import engine
from ..clustering import AHC
from ..transforms import PCA, LNorm


class DiarAHCPLDA:
    """Diarization of one recording by clustering its segments on PLDA scores
    (hyperion/diarization/diar_ahc_plda.py:21-168): pre-processing, optionally a PCA fitted on the
    recording with the PLDA model projected onto it, the [segments x segments] self-score matrix,
    average-linkage AHC cut at `threshold`.  The vectors, the PCA moments and the score matrix are
    device work; the eigendecomposition, the model projection and the linkage are host work on
    small matrices.  With do_unsup_cal a two-Gaussian mixture with one shared variance is fitted to
    the scores above the diagonal (on the device); with use_bic a recording whose scores one
    Gaussian explains as well (negative BIC) comes back as a single cluster.  As in the reference,
    the calibrated scores themselves do not reach the clustering (there they replace the scores
    only when a histogram plot is asked for, diar_ahc_plda.py:151-154; plots are not made here)."""

    def __init__(self, plda_model, preproc=None, threshold=0, pca_var_r=1, do_unsup_cal=False, use_bic=False):
        self.plda_model = plda_model
        self.preproc = preproc
        self.threshold = threshold
        self.pca_var_r = pca_var_r
        self.do_unsup_cal = do_unsup_cal
        self.use_bic = use_bic and do_unsup_cal
        self._ahc = AHC()

    @staticmethod
    def _unsup_gmm_calibration(scores, var_floor=1e-3, epochs=20):
        """Unsupervised calibration of a self-score matrix (diar_ahc_plda.py:100-120): the scores
        above the diagonal are modelled by two Gaussians with one shared variance, started from the
        single Gaussian of all scores split at mean +- one deviation and trained by EM
        (hyperion/pdfs/mixtures/gmm_tied_diag_cov.py:53-121: component variances floored at
        var_floor times their mean, then pooled).  The log-likelihood ratio of the two components
        is linear in the score: returns (scale * scores + bias, bic, (pi, mu, Lambda)), bic being
        the mean log-likelihood gain of two Gaussians over one minus the penalty of the four extra
        parameters.  Device float64 throughout; `scores` may be a host array or a device tensor
        (the result is of the same kind)."""
        import math

        torch = engine.require_gpu()
        is_dev = isinstance(scores, torch.Tensor)
        S = scores.to(device="cuda", dtype=torch.float64) if is_dev else torch.from_numpy(
            np.ascontiguousarray(scores, dtype=np.float64)).cuda()
        n_all = S.shape[0]
        iu = torch.triu_indices(n_all, n_all, offset=1, device=S.device)
        x = S[iu[0], iu[1]]
        n = x.numel()
        assert n >= 1, "calibration needs at least two segments"
        m1 = x.mean()
        lam1 = 1.0 / ((x - m1) ** 2).mean()
        half_log_2pi = 0.5 * math.log(2 * math.pi)

        def comp_llk(pi, mu, lam):
            return torch.log(pi) + 0.5 * torch.log(lam) - half_log_2pi - 0.5 * lam * (x[:, None] - mu) ** 2

        def log_prob(pi, mu, lam):
            r = comp_llk(pi, mu, lam)
            mx = r.max(dim=-1, keepdim=True).values
            return torch.log(torch.exp(r - mx).sum(dim=-1) + 1e-20) + mx[:, 0]

        sd = 1.0 / torch.sqrt(lam1)
        pi = torch.full((2,), 0.5, dtype=torch.float64, device=S.device)
        mu = torch.stack((m1 + sd, m1 - sd))
        lam = lam1
        for _ in range(epochs):
            z = torch.softmax(comp_llk(pi, mu, lam), dim=-1)
            N = z.sum(dim=0)
            mu = (z.T @ x) / N
            var = (z.T @ (x * x)) / N - mu * mu
            var = torch.maximum(var, var_floor * var.mean())
            lam = 1.0 / ((N * var).sum() / N.sum())
            pi = N / N.sum()
        one = torch.ones((1,), dtype=torch.float64, device=S.device)
        bic = float((log_prob(pi, mu, lam) - log_prob(one, m1[None], lam1)).mean().item()) \
            - 4 * math.log(n) / 2 / n
        scale = (mu[0] - mu[1]) * lam
        bias = (mu[1] ** 2 - mu[0] ** 2) * lam / 2 + torch.log(pi[0]) - torch.log(pi[1])
        cal = scale * S + bias
        gmm = (pi.cpu().numpy(), mu.cpu().numpy(), float(lam.item()))
        return (cal.to(scores.dtype) if is_dev else cal.cpu().numpy()), bic, gmm

    def scores(self, x):
        """The self-score matrix the clustering works on, as a device tensor [n, n]."""
        x = engine.upload(x)
        if self.preproc is not None:
            x = self.preproc.predict(x)
        plda_model = self.plda_model
        if self.pca_var_r < 1:
            pca = PCA(pca_var_r=self.pca_var_r, whiten=True)
            pca.fit(x)
            x = LNorm().predict(pca.predict(x))
            plda_model = plda_model.project(pca.T, pca.mu)
        return plda_model.llr_1vs1(x, x, refine=True)

    @staticmethod
    @engine.small_host_algebra
    def _recording_models(C, F, sizes, plda_model, pca_var_r):
        """The PCA of every recording from its moments (host float64 [E, d, d], [E, d]) and the model projected
        onto it, as padded parameters of three device steps: (W1, b1, dims) of the projection, (W2, b2) of the
        model's basis, (maps, c) of the packing."""
        E, d = F.shape
        firsts, folds = [], []
        for e in range(E):
            mu = F[e] / sizes[e]
            pca = PCA(pca_var_r=pca_var_r, whiten=True)
            pca.fit(mu=mu, S=C[e] / sizes[e] - np.outer(mu, mu))
            model = plda_model.project(pca.T, pca.mu)
            model._validate_for_scoring()
            firsts.append((pca.T, -(pca.mu @ pca.T)))
            folds.append((model._shared_fold(), float(model._fold()[4])))
        dims = np.array([T.shape[1] for T, _ in firsts])
        D, K = int(dims.max()), folds[0][0]["P"].shape[1]
        W1, b1 = np.zeros((E, d, D), np.float32), np.zeros((E, D), np.float32)
        W2, b2 = np.zeros((E, D, K), np.float32), np.zeros((E, K), np.float32)
        maps, c = np.zeros((E, 4, K), np.float32), np.zeros(E, np.float32)
        for e, ((T, b), (f, ce)) in enumerate(zip(firsts, folds)):
            k = dims[e]
            W1[e, :, :k], b1[e, :k] = T, b
            W2[e, :k], b2[e] = f["P"], f["pb"]
            maps[e] = f["shift_t"], f["scale_t"], f["shift_n"], f["scale_n"]
            c[e] = ce
        return W1, b1, dims, W2, b2, maps, c

    def scores_batch(self, xs):
        """Self-score matrices of a batch of recordings, each [segments, dim]: a list of device tensors
        [n, n].  The steps of `scores` (without its float64 refinement: entries that cancel
        to about zero carry an absolute error of some 1e-6 of the terms they are the difference of), every step
        one launch over all recordings: moments, projection with length normalisation, model basis, packing and
        the blocks of scores (one launch per recording above 510 latent dimensions, where packed rows are wider than
        the grouped product takes).  A recording needs two segments where a PCA is fitted on it."""
        torch = engine.require_gpu()
        xs = [engine.upload(x) for x in xs]
        if not xs:
            return []
        if len({x.shape[1] for x in xs}) != 1:
            raise ValueError("the recordings have vectors of different dimensions")
        sizes = [int(x.shape[0]) for x in xs]
        x = engine.upload(torch.cat(xs))
        if self.preproc is not None:
            x = self.preproc.predict(x)
        groups = engine.RowGroups(sizes)
        pairs = engine.GroupPairs(groups, groups)
        if self.pca_var_r < 1:
            if min(sizes) < 2:
                raise ValueError("a PCA needs recordings of at least two segments")
            C, F = engine.grouped_gram64(x, groups)
            W1, b1, dims, W2, b2, maps, c = self._recording_models(C.cpu().numpy(), F.cpu().numpy(), sizes,
                                                                  self.plda_model, self.pca_var_r)
            z = engine.grouped_affine(x, groups, engine.AffineBank(W1, b1, dims=dims), lnorm=True)
            s = engine.grouped_affine(z, groups, engine.AffineBank(W2, b2))
            G1, G2 = engine.grouped_pack(s, groups, maps, c)
        else:
            plan = self.plda_model.score_plan()
            G1, G2 = plan.prologue(x, engine.SIDE_ENROL), plan.prologue(x, engine.SIDE_TEST)
        if not engine.grouped_score_supported(G1.shape[1]):
            at = groups.offsets
            return [engine.score(G1[a:b], G2[a:b]) for a, b in zip(at[:-1], at[1:])]
        return pairs.blocks(engine.grouped_score(G1, G2, pairs))

    def cluster_batch(self, xs):
        """`cluster` for a batch of recordings, scored together (scores_batch): a list of cluster ids per segment.
        A recording of fewer than two segments is one cluster."""
        xs = list(xs)
        many = [i for i, x in enumerate(xs) if x.shape[0] > 1]
        ids = [np.zeros(x.shape[0], dtype=int) for x in xs]
        for i, scores in zip(many, self.scores_batch([xs[i] for i in many])):
            ids[i] = self._cluster_scores(scores)
        return ids

    def cluster(self, x, hist_file=None):
        """x [segments, dim] -> cluster id per segment (host int array).  hist_file (a plot in the
        reference) is ignored."""
        return self._cluster_scores(self.scores(x))

    def _cluster_scores(self, scores):
        if self.do_unsup_cal:
            _, bic, _ = self._unsup_gmm_calibration(scores)
            if self.use_bic and bic < 0:  # one Gaussian is enough: target trials only
                return np.zeros(scores.shape[0], dtype=int)
        self._ahc.fit(scores)
        return self._ahc.get_flat_clusters(self.threshold)

    @staticmethod
    def filter_args(**kwargs):
        valid = ("threshold", "pca_var_r", "do_unsup_cal", "use_bic")
        return {k: kwargs[k] for k in valid if k in kwargs}

    @staticmethod
    def add_class_args(parser, prefix=None):
        """hyperion/diarization/diar_ahc_plda.py:186-203."""
        p1 = "--" if prefix is None else "--" + prefix + "."
        parser.add_argument(p1 + "threshold", default=0, type=float)
        parser.add_argument(p1 + "pca-var-r", default=1, type=float)
        parser.add_argument(p1 + "do-unsup-cal", default=False, action="store_true")
        parser.add_argument(p1 + "use-bic", default=False, action="store_true")

    add_argparse_args = add_class_args
