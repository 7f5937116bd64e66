"""Plans of the grouped operators that are used on another stream than their own: their storage is marked as used there,
and memory of a dropped plan is not handed out while a launch still reads it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class _Storage:
    """Stands for a tensor in a plan's list of storage and notes the streams it is marked for."""

    def __init__(self):
        self.streams = []

    def record_stream(self, stream):
        self.streams.append(stream.cuda_stream)


def test_every_plan_of_a_call_is_marked_on_another_stream():
    import torch

    from hyperion_amd import engine

    r = np.random.RandomState(0)
    sizes = [5, 0, 9]
    rows, cols = engine.RowGroups(sizes), engine.RowGroups([4, 2, 8])
    pairs = engine.GroupPairs(rows, cols)
    bank = engine.AffineBank(r.randn(3, 6, 8))
    x = torch.from_numpy(r.randn(14, 6)).float().cuda()
    maps, c = torch.zeros(3, 4, 6, device="cuda"), torch.zeros(3, device="cuda")
    G1, G2 = torch.ones(14, 40, device="cuda"), torch.ones(14, 40, device="cuda")
    gallery = engine.q4_rows(G2, 30, cols)
    torch.cuda.synchronize()
    calls = (((rows, bank), lambda: engine.grouped_affine(x, rows, bank)),
             ((rows,), lambda: engine.grouped_gram64(x, rows)),
             ((rows,), lambda: engine.grouped_pack(x, rows, maps, c)),
             ((rows, cols, pairs), lambda: engine.grouped_score(G1, G2, pairs)),
             ((cols,), lambda: engine.q4_rows(G2, 30, cols)),
             ((rows, cols, pairs, gallery), lambda: engine.q4_score(gallery, G1, pairs)))
    other = torch.cuda.Stream()
    for plans, call in calls:
        kept = [p._storage for p in plans]
        for p, storage in zip(plans, kept):
            assert len(storage) >= 1 and all(isinstance(t, torch.Tensor) for t in storage)
            p._storage = [_Storage() for _ in storage]
        call()  # on the stream they were made on
        assert all(s.streams == [] for p in plans for s in p._storage)
        with torch.cuda.stream(other):
            call()
        assert all(s.streams and set(s.streams) == {other.cuda_stream} for p in plans for s in p._storage)
        for p, storage in zip(plans, kept):
            p._storage = storage
    torch.cuda.synchronize()
    held = {t.data_ptr() for p in (rows, pairs, bank, gallery) for t in p._storage}
    assert {rows._rows[0], pairs._rows[0], bank._w.data_ptr(), bank._c.data_ptr(), gallery.codes.data_ptr(),
            gallery.scales.data_ptr(), gallery.q.data_ptr()} <= held


def test_storage_of_a_dropped_plan_waits_for_the_launch_that_reads_it():
    """Maps and a gallery made on the default stream, used behind some milliseconds of work on another and dropped; then
    the default stream fills many blocks of exactly their sizes with zeros."""
    import torch

    from hyperion_amd import engine

    sizes = [40, 0, 1, 300, 77]
    groups = engine.RowGroups(sizes)
    pairs = engine.GroupPairs(groups, groups)
    other = torch.cuda.Stream()

    def make(seed):
        r = np.random.RandomState(seed)
        bank = engine.AffineBank(r.randn(5, 60, 30) / 8, r.randn(5, 30))
        G = torch.from_numpy(r.randn(418, 32)).float().cuda()
        x = torch.from_numpy(r.randn(418, 60)).float().cuda()
        torch.cuda.synchronize()
        return bank, engine.q4_rows(G, 30, groups), G, x

    for seed in range(4):
        bank, gallery, G, x = make(seed)
        want = [engine.grouped_affine(x, groups, bank), engine.q4_score(gallery, G, pairs)]
        torch.cuda.synchronize()
        shapes = [(t.shape, t.dtype) for t in bank._storage + gallery._storage]
        with torch.cuda.stream(other):
            busy = torch.ones(4096, 4096, device="cuda")
            for _ in range(20):
                busy = busy @ busy * 1e-4
            got = [engine.grouped_affine(x, groups, bank), engine.q4_score(gallery, G, pairs)]
        del bank, gallery
        filled = [torch.zeros(s, dtype=t, device="cuda") for _ in range(16) for s, t in shapes]
        torch.cuda.synchronize()
        assert len(filled) == 80 and all(torch.equal(a, b) for a, b in zip(got, want))
