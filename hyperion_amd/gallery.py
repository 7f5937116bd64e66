"""Identification of a few vectors among many enrolled ones: PLDA scores against a gallery held in 4 bits."""
import numpy as np

from . import engine
from .engine import SIDE_ENROL, SIDE_TEST
from .hyp_defs import float_cpu


# Scores that identify holds at a time: 1000 tests against a million rows take 12.2 ms, in slices of 1 GiB 13.3
_SLICE_BYTES = 4 << 30


class PLDAGallery:
    """Enrolled vectors as 4-bit rows (engine.q4_rows: 94 bytes a row at y_dim 150, a sixth of the packed fp32 row),
    scored against test vectors in one pass over them.  plda: an SPLDA, FRPLDA or PLDA model of up to 512 latent
    dimensions; preproc: a TransformList folded in front of it, as in PLDABackend.

    The scores are llr_1vs1 (hyperion/pdfs/plda/splda.py:275-316) with the enrolled projections rounded to 4 bits: a
    score is off by at most half a scale per coordinate times the test's projection, about a tenth of the deviation
    of non-target scores at y_dim 150.  They rank candidates; what is decided on them is scored again with
    llr_1vs1 on the few that are left.

    Enrolled vectors can be kept in partitions (per site, language or customer): a test vector is then scored against
    its own partition alone."""

    def __init__(self, plda, preproc=None):
        self.plda = plda
        self.plan = plda.score_plan(preproc)
        if not engine.q4_supported(self.plan.k):
            raise ValueError("a gallery holds models of up to 512 latent dimensions, this one has %d" % self.plan.k)
        # (4-bit rows, device int64: row of the enrolled array that each was made from), replaced together
        self._enrolled = None, None

    @property
    def gallery(self):
        return self._enrolled[0]

    @property
    def rows(self):
        return self._enrolled[1]

    def enrol(self, x, partition=None, num_partitions=None):
        """Replaces the gallery by the vectors x [n, d] (host array or device tensor); partition: number of every
        vector's partition, 0 .. num_partitions - 1.  Waits until the gallery is written, so that any stream can search it at
        once.  Returns self."""
        torch = engine.require_gpu()
        if partition is None and num_partitions not in (None, 1):
            raise ValueError("%d partitions: say which one every vector belongs to" % num_partitions)
        x = engine.upload(x)
        if partition is None:
            groups, order = engine.RowGroups([x.shape[0]], device=x.device), None
        else:
            if len(partition) != x.shape[0]:
                raise ValueError("%d partition numbers for %d vectors" % (len(partition), x.shape[0]))
            g = engine.RowGroups.from_ids(partition, num_partitions, device=x.device)
            groups, order = engine.RowGroups(g.sizes, device=x.device), g.order.long()
        G = self.plan.prologue(x, SIDE_ENROL)
        rows = torch.arange(x.shape[0], device=x.device) if order is None else order
        gallery = engine.q4_rows(G if order is None else G[order], self.plan.k, groups)
        torch.cuda.current_stream(x.device).synchronize()
        self._enrolled = gallery, rows
        return self

    def _tests(self, x, partition):
        """(4-bit rows, rows of the enrolled array, test vectors per partition, rows of x in the order of the partitions
        or None, packed test rows in that order)."""
        gallery, rows = self._enrolled
        if gallery is None:
            raise ValueError("nothing is enrolled")
        x = engine.upload(x)
        # a concurrent enrol may drop the rows while this stream reads them
        rows.record_stream(engine.require_gpu().cuda.current_stream(rows.device))
        groups, order, sizes = gallery.groups, None, np.array([x.shape[0]])
        if partition is None:
            if groups.num_groups != 1:
                raise ValueError("the gallery has %d partitions: say which one every test vector belongs to"
                                 % groups.num_groups)
        else:
            if len(partition) != x.shape[0]:
                raise ValueError("%d partition numbers for %d vectors" % (len(partition), x.shape[0]))
            g = engine.RowGroups.from_ids(partition, groups.num_groups, device=x.device)
            sizes, order = g.sizes, g.order.long()
        G = self.plan.prologue(x, SIDE_TEST)
        return gallery, rows, sizes, order, G if order is None else G[order]

    @staticmethod
    def _score(gallery, sizes, G):
        pairs = engine.GroupPairs(engine.RowGroups(sizes, device=G.device), gallery.groups)
        return pairs, engine.q4_score(gallery, G, pairs)

    def _best(self, gallery, enrolled, part, G, at, rows, best):
        """The best enrolled vectors of the packed tests G, ascending by partition, into the rows `at` of the result."""
        torch = engine.require_gpu()
        pairs, flat = self._score(gallery, np.bincount(part, minlength=gallery.groups.num_groups), G)
        flat.masked_fill_(torch.isnan(flat), -np.inf)
        for e in np.unique(part):
            blk = pairs.block(flat, e)
            if blk.numel() == 0:
                continue
            k = min(best.shape[1], blk.shape[1])
            s, i = torch.topk(blk, k, dim=1)
            to = at[int(pairs.rows.offsets[e]):int(pairs.rows.offsets[e + 1])]
            best[to, :k] = s
            rows[to, :k] = torch.where(torch.isinf(s) & (s < 0), -1, enrolled[int(pairs.cols.offsets[e]) + i])

    def llr(self, x, partition=None):
        """Scores of the test vectors x [m, d].  Without partitions [n, m], enrolled vectors by test vectors, as
        llr_1vs1 returns them (host array for a host array, device tensor for a device tensor).  With partitions a
        list of (rows of the enrolled array, rows of x, [rows, tests] scores), one per partition."""
        torch = engine.require_gpu()
        is_dev = isinstance(x, torch.Tensor)
        gallery, enrolled, sizes, order, G = self._tests(x, partition)
        pairs, flat = self._score(gallery, sizes, G)

        def host(t):
            return t if is_dev else t.cpu().numpy() if t.dtype == torch.int64 else engine.to_host(t, float_cpu())

        if partition is None:
            return host(pairs.block(flat, 0).t())
        res = []
        for e in range(pairs.rows.num_groups):
            g, t = pairs.cols.offsets, pairs.rows.offsets
            res.append((host(enrolled[g[e]:g[e + 1]]), host(order[t[e]:t[e + 1]]), host(pairs.block(flat, e).t())))
        return res

    def identify(self, x, nbest=10, partition=None):
        """The nbest enrolled vectors of every test vector: (rows of the enrolled array [m, nbest], scores
        [m, nbest]), best first, host arrays for a host array.  Where fewer are enrolled the rest is row -1 with
        score -inf; vectors whose score is NaN are never named.  Scores are held 4 GiB at a time."""
        torch = engine.require_gpu()
        is_dev = isinstance(x, torch.Tensor)
        if nbest < 1:
            raise ValueError("nbest must be at least 1")
        gallery, enrolled, sizes, order, G = self._tests(x, partition)
        m = G.shape[0]
        rows = torch.full((m, nbest), -1, dtype=torch.int64, device=G.device)
        best = torch.full((m, nbest), -np.inf, dtype=torch.float32, device=G.device)
        part = np.repeat(np.arange(len(sizes)), sizes)  # of every test, in the order of G
        scores = np.concatenate([[0], np.cumsum(gallery.groups.sizes[part])])  # of the tests before each
        start = 0
        while start < m:  # as many tests as a slice has room for the scores of, at least one
            end = max(start + 1, int(np.searchsorted(scores, scores[start] + _SLICE_BYTES // 4, side="right")) - 1)
            at = torch.arange(start, end, device=G.device) if order is None else order[start:end]
            self._best(gallery, enrolled, part[start:end], G[start:end], at, rows, best)
            start = end
        return (rows, best) if is_dev else (rows.cpu().numpy(), best.cpu().numpy().astype(float_cpu(), copy=False))
