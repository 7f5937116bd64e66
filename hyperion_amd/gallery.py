"""Identification of a few vectors among many enrolled ones: PLDA scores against a gallery held in 4 bits."""
import numpy as np

from . import engine
from .engine import SIDE_ENROL, SIDE_TEST
from .hyp_defs import float_cpu


class PLDAGallery:
    """Enrolled vectors as 4-bit rows (engine.q4_rows: 94 bytes a row at y_dim 150, a sixth of the packed fp32 row),
    scored against test vectors in one pass over them.  plda: an SPLDA, FRPLDA or PLDA model; preproc: a
    TransformList folded in front of it, as in PLDABackend.

    The scores are llr_1vs1 (hyperion/pdfs/plda/splda.py:275-316) with the enrolled projections rounded to 4 bits: a
    score is off by at most half a scale per coordinate times the test's projection, about a tenth of the deviation
    of non-target scores at y_dim 150.  They rank candidates; what is decided on them is scored again with
    llr_1vs1 on the few that are left.

    Enrolled vectors can be kept in partitions (per site, language or customer): a test vector is then scored against
    its own partition alone."""

    def __init__(self, plda, preproc=None):
        self.plda = plda
        self.plan = plda.score_plan(preproc)
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

    def _score(self, x, partition):
        gallery, rows = self._enrolled
        if gallery is None:
            raise ValueError("nothing is enrolled")
        x = engine.upload(x)
        # a concurrent enrol may drop the rows while this stream reads them
        rows.record_stream(engine.require_gpu().cuda.current_stream(rows.device))
        groups, order = gallery.groups, None
        if partition is None:
            if groups.num_groups != 1:
                raise ValueError("the gallery has %d partitions: say which one every test vector belongs to"
                                 % groups.num_groups)
            tests = engine.RowGroups([x.shape[0]], device=x.device)
        else:
            if len(partition) != x.shape[0]:
                raise ValueError("%d partition numbers for %d vectors" % (len(partition), x.shape[0]))
            g = engine.RowGroups.from_ids(partition, groups.num_groups, device=x.device)
            tests, order = engine.RowGroups(g.sizes, device=x.device), g.order.long()
        G = self.plan.prologue(x, SIDE_TEST)
        pairs = engine.GroupPairs(tests, groups)
        return pairs, order, rows, engine.q4_score(gallery, G if order is None else G[order], pairs)

    def llr(self, x, partition=None):
        """Scores of the test vectors x [m, d].  Without partitions [n, m], enrolled vectors by test vectors, as
        llr_1vs1 returns them (host array for a host array, device tensor for a device tensor).  With partitions a
        list of (rows of the enrolled array, rows of x, [rows, tests] scores), one per partition."""
        torch = engine.require_gpu()
        is_dev = isinstance(x, torch.Tensor)
        pairs, order, enrolled, flat = self._score(x, partition)

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
        score -inf; vectors whose score is NaN are never named."""
        torch = engine.require_gpu()
        is_dev = isinstance(x, torch.Tensor)
        if nbest < 1:
            raise ValueError("nbest must be at least 1")
        pairs, order, enrolled, flat = self._score(x, partition)
        m = pairs.rows.total
        rows = torch.full((m, nbest), -1, dtype=torch.int64, device=flat.device)
        best = torch.full((m, nbest), -np.inf, dtype=torch.float32, device=flat.device)
        flat = torch.where(torch.isnan(flat), -np.inf, flat)
        for e in range(pairs.rows.num_groups):
            blk = pairs.block(flat, e)
            k = min(nbest, blk.shape[1])
            if blk.numel() == 0:
                continue
            s, i = torch.topk(blk, k, dim=1)
            t0, t1 = int(pairs.rows.offsets[e]), int(pairs.rows.offsets[e + 1])
            at = slice(t0, t1) if order is None else order[t0:t1]
            best[at, :k] = s
            rows[at, :k] = torch.where(torch.isinf(s) & (s < 0), -1, enrolled[int(pairs.cols.offsets[e]) + i])
        return (rows, best) if is_dev else (rows.cpu().numpy(), best.cpu().numpy().astype(float_cpu(), copy=False))
