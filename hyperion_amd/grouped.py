"""Grouped operators: rows that fall into groups of unequal sizes (the recordings of a batch, the domains
of a trial set, the partitions of a gallery), each group with its own matrix, its own moments or its own
block of scores, in one launch.  The names here are part of hyperion_amd.engine.

A batch is described once, by a RowGroups (sizes on the host, tables on the device) and, for products of
two sides, a GroupPairs; on device tensors the operators themselves neither wait for the device nor send it anything,
so they can be captured in a HIP graph.  Inputs have to be on one device; the work runs on that device's current
stream.  A RowGroups, a GroupPairs and an AffineBank are complete when they have been made (which waits for the
current stream) and can be used on any stream at once; a Q4Rows is filled by a launch on the stream it is made on, for
which another stream waits as for any tensor."""
import numpy as np

from . import _lib
from .engine import _ptr, _torch, require_gpu, round_up

_AFFINE_TILES = (16, 64, 128)
_Q4_TESTS = (16, 32, 64)


def _affine_tile(mean, d_in, itemsize):
    """Rows per workgroup of the affine map, by the mean size of the groups.  Measured with 200 groups of ragged
    sizes, tiles of 16 / 64 / 128 rows in us.  Small groups: fp32 200 -> 200 with 12 rows a group 10.7 / 12.4 / 18,
    with 24 rows 15.2 / 13.3 / 19; 512 -> 200 18.6 / 20.6 / 33 and 22.4 / 21.3 / 33.  Large ones, tiles of 64 / 128:
    fp32 512 -> 200 with 200 rows 44 / 50, with 870 rows 42 / 49; 512 -> 150 with 5600 rows 144 / 160; 96 -> 64 with
    32 000 rows 20.5 / 19.3, which has few coordinates to overlap with what starts and ends a tile.  Rows of 16 bits
    are less work to convert and take the larger tile, which reads the weights half as often: bf16 512 -> 150 with 400 rows
    76 / 90, with 1500 rows 59 / 56; 512 -> 200 with 19 000 rows 114 / 107."""
    if mean <= 20:
        return 16
    return 128 if mean > 1000 and (itemsize == 2 or d_in <= 128) else 64


def _prefix(counts):
    out = np.zeros(len(counts) + 1, dtype=np.int64)
    np.cumsum(counts, out=out[1:])
    return out


def _ceil(a, b):
    return -(-a // b)


def _device(device=None):
    torch = require_gpu()
    d = torch.device("cuda" if device is None else device)
    if d.type != "cuda":
        raise ValueError("the grouped operators work on the GPU, not on %s" % d)
    return torch.device("cuda", torch.cuda.current_device() if d.index is None else d.index)


def _tables(arrays, device):
    """Host int64 tables of equal length as rows of one device tensor (one copy, complete on return)."""
    torch = _torch()
    return torch.from_numpy(np.ascontiguousarray(np.stack(arrays))).to(device)


def _run(fn, device, owners, *args):
    """Calls the library function `fn` with `args` and the current stream of `device`.  owners: the plans whose
    storage the launch reads; on another stream than the one they were made on their storage is marked as used
    there, so that dropping a plan does not hand its memory to someone else while the launch is running."""
    torch = _torch()
    index = device.index
    raw = torch._C._cuda_getCurrentRawStream(index)
    for o in owners:
        if o._stream != raw:
            stream = torch.cuda.current_stream(device)
            for t in o._storage:
                t.record_stream(stream)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, raw)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, raw)
    if rc:
        _lib.check(rc)


class _Plan:
    """Device storage that is made once and read by many launches."""

    def _own(self, *tensors):
        self._storage = [t for t in tensors if t is not None]
        self._stream = _torch()._C._cuda_getCurrentRawStream(self.device.index)


class RowGroups(_Plan):
    """Rows in groups: group e owns `sizes[e]` consecutive rows (zero is allowed), in order, or, with
    `order`, the rows order[offsets[e]] .. order[offsets[e + 1] - 1]; every row may be listed once.
    sizes: host integers.  order: host or device integers, one per listed row."""

    def __init__(self, sizes, order=None, device=None):
        sizes = np.asarray(sizes)
        if sizes.ndim != 1 or (sizes.size and sizes.dtype.kind not in "iu"):
            raise ValueError("group sizes must be a 1-D sequence of integers")
        if sizes.size > 1 << 30:  # the search for a row's group counts in 32 bits, with some steps to spare
            raise ValueError("at most 2^30 groups")
        sizes = sizes.astype(np.int64)
        if sizes.size and sizes.min() < 0:
            raise ValueError("group sizes must not be negative")
        if sizes.sum(dtype=np.float64) > 2.0 ** 40:
            raise ValueError("at most 2^40 rows")
        self.sizes = sizes
        self.offsets = _prefix(sizes)
        self.num_groups = int(sizes.size)
        self.total = int(self.offsets[-1])
        self.device = _device(device)
        self.order = None
        self.num_rows = self.total  # rows an input needs at least
        if order is not None:
            self._set_order(order)
        lib = _lib.load()
        span, split = lib.hypmi_grouped_gram_span(), lib.hypmi_grouped_gram_split()
        cut = _ceil(sizes, span)
        # chunks of one length; the last may be short
        rest = sizes - (np.maximum(cut, 1) - 1) * round_up(_ceil(sizes, np.maximum(cut, 1)), 64)
        prefix = [_prefix(_ceil(sizes, t)) for t in _AFFINE_TILES]
        units = _prefix(4 * (np.maximum(cut, 1) - 1) + np.where(rest > split, 4, 1))
        slots = _prefix(np.where(cut > 1, cut, 0))
        self._tab = _tables([self.offsets] + prefix + [units, slots], self.device)
        base = self._tab.data_ptr()
        self._rows = [base + 8 * i * (self.num_groups + 1) for i in range(6)]  # device pointers of the tables
        self._n_tiles = dict(zip(_AFFINE_TILES, (int(p[-1]) for p in prefix)))
        self._n_units, self._n_slots = int(units[-1]), int(slots[-1])
        self._order_ptr = None if self.order is None else self.order.data_ptr()
        self._mean = self.total / max(1, int(np.count_nonzero(sizes)))
        self._own(self._tab, self.order)

    @classmethod
    def from_ids(cls, ids, num_groups=None, device=None):
        """Groups of rows by a group number per row, 0 .. num_groups - 1 (default: the largest + 1)."""
        ids = np.asarray(ids)
        if ids.ndim != 1 or (ids.size and ids.dtype.kind not in "iu"):
            raise ValueError("group ids must be a 1-D sequence of integers")
        ids = ids.astype(np.int64)
        top = int(ids.max()) + 1 if ids.size else 0
        if num_groups is None:
            num_groups = top
        if ids.size and (ids.min() < 0 or top > num_groups):
            raise ValueError("group ids must lie in 0 .. %d" % (num_groups - 1))
        return cls(np.bincount(ids, minlength=num_groups), np.argsort(ids, kind="stable"), device)

    def _set_order(self, order):
        torch = _torch()
        if not isinstance(order, torch.Tensor):
            order = np.ascontiguousarray(order)
            order = torch.from_numpy(order if order.size else order.astype(np.int64))  # an empty list has no type
        if order.dim() != 1 or order.dtype not in (torch.int32, torch.int64):
            raise ValueError("order must be a 1-D sequence of integers")
        if order.numel() != self.total:
            raise ValueError("order lists %d rows, the groups hold %d" % (order.numel(), self.total))
        if self.total:
            lo, hi = int(order.min()), int(order.max())
            if lo < 0 or hi > 0x7fffffff:
                raise ValueError("order must hold row numbers from 0 to 2^31 - 1")
            self.num_rows = hi + 1
        # a copy: what the caller does to its tensor later must not reach a launch
        self.order = torch.empty(self.total, dtype=torch.int32, device=self.device).copy_(order)
        if self.total:
            seen = torch.zeros(hi + 1, dtype=torch.int8, device=self.device)
            seen[self.order.long()] = 1
            if int(seen.sum(dtype=torch.int64)) != self.total:  # waits, for the copy too
                raise ValueError("order lists a row more than once")

    def _check(self, x, what):
        if x.get_device() != self.device.index:
            raise ValueError("%s is on %s, its groups are on %s" % (what, x.device, self.device))
        if self.order is None:
            if x.shape[0] != self.total:
                raise ValueError("%s has %d rows, its groups hold %d" % (what, x.shape[0], self.total))
        elif x.shape[0] < self.num_rows:
            raise ValueError("%s has %d rows, the order names row %d" % (what, x.shape[0], self.num_rows - 1))


class GroupPairs(_Plan):
    """Blocks of scores of two sides that have the same groups: block e is rows.sizes[e] x cols.sizes[e],
    the blocks lie one after the other in a flat result without padding."""

    def __init__(self, rows, cols):
        if rows.num_groups != cols.num_groups:
            raise ValueError("the two sides have %d and %d groups" % (rows.num_groups, cols.num_groups))
        if rows.device != cols.device:
            raise ValueError("the two sides are on %s and %s" % (rows.device, cols.device))
        if rows.order is not None or cols.order is not None:
            raise ValueError("score blocks need rows in group order (RowGroups without order)")
        self.rows, self.cols = rows, cols
        self.device = rows.device
        n1, n2 = rows.sizes, cols.sizes
        if np.sum(n1.astype(np.float64) * n2) > 2.0 ** 52:
            raise ValueError("at most 2^52 scores")
        self.offsets = _prefix(n1 * n2)
        self.numel = int(self.offsets[-1])
        lib = _lib.load()
        span = lib.hypmi_grouped_score_span()
        # tests per gallery task: unpacking the codes of a row costs as much as multiplying them with 7 tests, and a
        # tile is paid in full.  Tiles of 64 leave two waves per SIMD and pay where groups have hundreds of tests: a
        # million rows x 1000 tests 1579 / 1345 / 1216 us with tiles of 16 / 32 / 64, x 64 tests 102.5 / 102.6 / 106;
        # 200 000 rows x 48 tests 21.5 / 22.0 / 27.3, x 24 tests 17.7 / 17.0 / 24.8.
        cost = [float(np.sum(n2 * _ceil(n1, t) * (7.0 + t))) for t in _Q4_TESTS[:2]]
        many = self.numel >= 200 * max(1, int(n2.sum()))
        self._q4_tests = 64 if many else _Q4_TESTS[int(np.argmin(cost))]
        # gallery rows per task: three workgroups on each of 256 CUs at once, or a whole number of such rounds.  Tiles of
        # 64 tests have two on a CU; rounds of 512 in place of 768 are no better there: 200 000 rows x 300 tests 82 -> 71 us,
        # 50 000 x 1000 (64 coordinates) 50 -> 43, but 20 000 x 4000 108 -> 120, 40 partitions x 400 177 -> 188, a million
        # x 1000 1215 -> 1217.
        work = int(np.sum(n2 * _ceil(n1, self._q4_tests)))
        rounds = max(1, _ceil(work, 768 * 4096))
        self._q4_rows = max(256, round_up(_ceil(work, 768 * rounds), 64))
        tabs = [_prefix(_ceil(n1, b) * _ceil(n2, span)) for b in (64, 128)]
        tabs.append(_prefix(_ceil(n1, self._q4_tests) * _ceil(n2, self._q4_rows)))
        self._n_tasks = [int(t[-1]) for t in tabs]
        self._tab = _tables([self.offsets] + tabs, self.device)
        base = self._tab.data_ptr()
        self._rows = [base + 8 * i * (rows.num_groups + 1) for i in range(4)]  # device pointers of the tables
        self._own(self._tab)

    def block(self, flat, e):
        """Block e of a flat result as a [rows, cols] view."""
        return flat[int(self.offsets[e]):int(self.offsets[e + 1])].view(int(self.rows.sizes[e]), int(self.cols.sizes[e]))

    def blocks(self, flat):
        return [self.block(flat, e) for e in range(self.rows.num_groups)]

    def _result(self, out, *inputs):
        torch = _torch()
        if out is None:
            return torch.empty(self.numel, dtype=torch.float32, device=self.device)
        if out.dtype != torch.float32 or out.device != self.device or out.dim() != 1 or out.numel() != self.numel \
                or not out.is_contiguous():
            raise ValueError("out must be a contiguous fp32 vector of %d elements on %s" % (self.numel, self.device))
        if any(_overlap(a, out) for a in inputs):
            raise ValueError("out must not share memory with the inputs")
        return out


class AffineBank(_Plan):
    """One affine map per group, x -> x W[e] + b[e], laid out for grouped_affine.  W [E, d_in, d_out] and b
    [E, d_out] (or None), host arrays or device tensors of any float type, taken as fp32.  dims
    [E] (optional): dimension of every map where they differ; W[e][:, dims[e]:] and b[e][dims[e]:] have to be
    zero, and the length normalisation scales to sqrt(dims[e]).  The maps are laid out by the time the constructor
    returns, so that any stream can use them at once; made while a HIP graph is captured they are part of the graph."""

    def __init__(self, W, b=None, dims=None, device=None):
        torch = _torch()
        if device is None and isinstance(W, torch.Tensor) and W.is_cuda:
            device = W.device
        self.device = _device(device)
        W = self._fp32(W)
        if W.dim() != 3 or 0 in W.shape[1:]:
            raise ValueError("W must be [groups, d_in, d_out], got %s" % (tuple(W.shape),))
        self.num_groups, self.d_in, self.d_out = (int(v) for v in W.shape)
        if b is not None:
            b = self._fp32(b)
            if tuple(b.shape) != (self.num_groups, self.d_out):
                raise ValueError("b must be [%d, %d], got %s" % (self.num_groups, self.d_out, tuple(b.shape)))
        self.dims = None
        if dims is not None:
            dims = np.asarray(dims)
            if dims.shape != (self.num_groups,) or dims.dtype.kind not in "iu" or \
                    (dims.size and (dims.min() < 1 or dims.max() > self.d_out)):
                raise ValueError("dims must be %d integers in 1 .. %d" % (self.num_groups, self.d_out))
            self.dims = torch.from_numpy(dims.astype(np.int32)).to(self.device)
            used = (W != 0).any(1) if b is None else (W != 0).any(1) | (b != 0)
            if bool((used & (torch.arange(self.d_out, device=self.device) >= self.dims[:, None])).any()):
                raise ValueError("W and b must be zero behind dims: those columns would enter the length normalisation")
        lib = _lib.load()
        args = (self.num_groups, self.d_in, self.d_out)
        self._w = torch.empty(lib.hypmi_grouped_weights_bytes(*args) // 4, dtype=torch.int32, device=self.device)
        self._c = torch.empty(lib.hypmi_grouped_columns_bytes(self.num_groups, self.d_out) // 4, dtype=torch.float32,
                              device=self.device)
        self._own(self._w, self._c, self.dims)
        self._dims_ptr = None if self.dims is None else self.dims.data_ptr()
        if self.num_groups:
            _run(lib.hypmi_grouped_weights, self.device, (), _ptr(W), None if b is None else _ptr(b), *args,
                 _ptr(self._w), _ptr(self._c))
        with torch.cuda.device(self.device):
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()

    def _fp32(self, a):
        torch = _torch()
        if not isinstance(a, torch.Tensor):
            a = torch.from_numpy(np.ascontiguousarray(a))
        if not a.is_floating_point():
            raise ValueError("weights must be floating-point numbers")
        return a.to(device=self.device, dtype=torch.float32).contiguous()


_KINDS = {}


def _kinds(op):
    """Element types an operator takes -> their numbers in the C ABI."""
    if not _KINDS:
        torch = _torch()
        _KINDS["affine"] = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
        _KINDS["gram"] = {torch.float32: _lib.F32, torch.float64: _lib.F64}
        _KINDS["rows"] = {torch.float32: _lib.F32}
    return _KINDS[op]


def _device_rows(x, types, what):
    """A 2-D device tensor of one of `types` with unit column stride, as it is; a view with other strides is
    copied.  Returns (x, leading dimension)."""
    if not isinstance(x, _torch().Tensor) or not x.is_cuda:
        raise ValueError("%s must be a device tensor" % what)
    if x.dim() != 2:
        raise ValueError("%s must be 2-D, got shape %s" % (what, tuple(x.shape)))
    if x.dtype not in types:
        raise ValueError("%s is %s, expected one of %s" % (what, x.dtype, ", ".join(str(t) for t in types)))
    n, d = x.shape
    ld, step = x.stride()
    if (d > 1 and step != 1) or (n > 1 and ld < d):
        x = x.contiguous()
        ld = d
    return x, (ld if n > 1 else d)


def grouped_affine(x, groups, bank, lnorm=False, out=None):
    """y_r = x_r W_e + b_e for every row r of group e, with lnorm followed by the length normalisation
    y <- sqrt(dim_e) y / (|y| + 1e-10).  x: device fp32, fp16 or bf16 [n, d_in]; returns device fp32
    [n, d_out].  The coordinates of a row count to 22 bits, or to 2^-42 of the largest magnitude of their row where
    that is more (fp16 rows are taken exactly), weights to 22 bits or 2^-48 of the largest of their column; sums are
    fp32.  With an ordered RowGroups row i of the result belongs to row i of x; rows of
    no group are zero in a new result and left alone in `out` (fp32, 16-byte aligned rows, also a view whose
    storage goes on behind a row)."""
    torch = _torch()
    kinds = _kinds("affine")
    x, ldx = _device_rows(x, kinds, "x")
    groups._check(x, "x")
    if bank.device != groups.device:
        raise ValueError("the maps are on %s, the groups on %s" % (bank.device, groups.device))
    if bank.num_groups != groups.num_groups:
        raise ValueError("%d maps for %d groups" % (bank.num_groups, groups.num_groups))
    if x.shape[1] != bank.d_in:
        raise ValueError("expected %d-dim vectors, got %d" % (bank.d_in, x.shape[1]))
    n, d = x.shape[0], bank.d_out
    ld = round_up(d, 4)
    if out is None:
        make = torch.empty if groups.total == n else torch.zeros
        y = make((n, ld), dtype=torch.float32, device=x.device)
    else:
        y = out
        if y.dtype != torch.float32 or y.device != x.device or tuple(y.shape) != (n, d) or \
                (d > 1 and y.stride(1) != 1) or y.data_ptr() % 16 or (n > 1 and (y.stride(0) % 4 or y.stride(0) < d)):
            raise ValueError("out must be fp32 [%d, %d] on %s with 16-byte aligned rows" % (n, d, x.device))
        if _overlap(x, y):
            raise ValueError("out must not share memory with x")
    tile = _affine_tile(groups._mean, bank.d_in, x.element_size())
    n_tiles = groups._n_tiles[tile]
    if n_tiles:
        _run(_lib.load().hypmi_grouped_affine, x.device, (groups, bank), x.data_ptr(), kinds[x.dtype], ldx, bank.d_in,
             groups._rows[0], groups._rows[1 + _AFFINE_TILES.index(tile)], tile, groups.num_groups, groups.total, n_tiles,
             groups._order_ptr, bank._w.data_ptr(), bank._c.data_ptr(), bank._dims_ptr, d, int(bool(lnorm)),
             y.data_ptr(), ld if out is None else (y.stride(0) if n > 1 else ld), ld if out is None else d)
    return (y if ld == d else y[:, :d]) if out is None else out


def _overlap(a, b):
    """Whether the storage ranges of two tensors meet."""
    def end(t):
        last = sum([(s - 1) * st for s, st in zip(t.shape, t.stride())])
        return t.data_ptr() + t.element_size() * (1 + last)

    return a.numel() > 0 and b.numel() > 0 and a.data_ptr() < end(b) and b.data_ptr() < end(a)


def _packed(G, groups, what):
    """Packed rows as the grouped kernels take them: fp32, 16-byte aligned rows."""
    G, ld = _device_rows(G, _kinds("rows"), what)
    groups._check(G, what)
    if G.data_ptr() % 16 or ld % 4:
        raise ValueError("%s must have 16-byte aligned rows" % what)
    return G, ld


def grouped_pack(s, groups, maps, c, sides="both"):
    """Packed rows of the projected rows s [n, K] (device fp32, in group order) by the maps of their group: maps
    [E, 4, K] = shift_t, scale_t, shift_n, scale_n, c [E] (host arrays are sent, which waits).  Returns (enrol-side, test-side) rows
    [n, kp]; sides "enrol" or "test": the other is None."""
    torch = _torch()
    s, ld = _device_rows(s, _kinds("rows"), "s")
    groups._check(s, "s")
    if groups.order is not None:
        raise ValueError("packing needs rows in group order (RowGroups without order)")
    if sides not in ("both", "enrol", "test"):
        raise ValueError("sides must be both, enrol or test")
    n, K = s.shape
    maps, c = (torch.as_tensor(a).to(device=s.device, dtype=torch.float32).contiguous() for a in (maps, c))
    if tuple(maps.shape) != (groups.num_groups, 4, K) or tuple(c.shape) != (groups.num_groups,):
        raise ValueError("maps must be [%d, 4, %d] and c [%d]" % (groups.num_groups, K, groups.num_groups))
    lib = _lib.load()
    kp = lib.hypmi_packed_width(K)
    G1, G2 = (torch.empty((n, kp), dtype=torch.float32, device=s.device) if sides in ("both", side) else None
              for side in ("enrol", "test"))
    if n:
        _run(lib.hypmi_grouped_pack, s.device, (groups,), s.data_ptr(), ld, K, groups._rows[0], groups.num_groups, n,
             maps.data_ptr(), c.data_ptr(), None if G1 is None else G1.data_ptr(),
             None if G2 is None else G2.data_ptr(), kp)
    return G1, G2


def grouped_score_supported(kp):
    """Whether grouped_score takes packed rows of kp elements (multiples of 8 up to 512)."""
    return bool(_lib.load().hypmi_grouped_score_rows(int(kp)))


def grouped_score(G1, G2, pairs, out=None):
    """Scores of packed enrol rows against packed test rows of the same group (Plan.prologue, both [n, kp]):
    the flat device fp32 result of `pairs` (pairs.block(flat, e) is the [n1, n2] block of group e).  An element of a
    row counts to 22 bits, or to 2^-39 of the largest magnitude of its row where that is more, as in score."""
    same = G2 is G1 and pairs.cols is pairs.rows  # self-scores: checked once
    G1, ld1 = _packed(G1, pairs.rows, "G1")
    G2, ld2 = (G1, ld1) if same else _packed(G2, pairs.cols, "G2")
    kp = G1.shape[1]
    if G2.shape[1] != kp:
        raise ValueError("packed widths differ: %d vs %d" % (kp, G2.shape[1]))
    lib = _lib.load()
    rows = lib.hypmi_grouped_score_rows(kp)
    if not rows:
        raise ValueError("packed width %d has no grouped kernel (multiples of 8 up to 512)" % kp)
    S = pairs._result(out, G1, G2)
    i = 1 if rows == 64 else 2
    if pairs.numel:
        _run(lib.hypmi_grouped_score, pairs.device, (pairs, pairs.rows, pairs.cols), G1.data_ptr(), ld1, G2.data_ptr(),
             ld2, kp, pairs.rows._rows[0], pairs.cols._rows[0], pairs._rows[0], pairs._rows[i], pairs.rows.num_groups,
             pairs._n_tasks[i - 1], S.data_ptr())
    return S


def grouped_gram64(x, groups, w=None):
    """(sum_r w_r x_r x_r^T, sum_r w_r x_r) of every group as device float64 tensors [E, d, d] and [E, d]; x
    device fp32 or float64 [n, d], w optional float64 weights per row of x."""
    torch = _torch()
    kinds = _kinds("gram")
    x, ldx = _device_rows(x, kinds, "x")
    groups._check(x, "x")
    d, E = x.shape[1], groups.num_groups
    if d < 1:
        raise ValueError("x has no columns")
    if w is not None:
        if not isinstance(w, torch.Tensor) or w.device != x.device or w.dtype != torch.float64 or \
                tuple(w.shape) != (x.shape[0],):
            raise ValueError("w must be a float64 vector of %d elements on %s" % (x.shape[0], x.device))
        w = w.contiguous()
    lib = _lib.load()
    C = torch.empty((E, d, d), dtype=torch.float64, device=x.device)
    F = torch.empty((E, d), dtype=torch.float64, device=x.device)
    nbytes = lib.hypmi_grouped_gram_workspace_bytes(groups._n_slots, d)
    ws = torch.empty(nbytes // 8, dtype=torch.float64, device=x.device) if nbytes else None
    if E:
        _run(lib.hypmi_grouped_gram_f64, x.device, (groups,), x.data_ptr(), kinds[x.dtype], ldx, d,
             None if w is None else w.data_ptr(), groups._rows[0], groups._rows[4], groups._rows[5], E, groups._n_units,
             groups._n_slots, groups._order_ptr, C.data_ptr(), F.data_ptr(), None if ws is None else ws.data_ptr(), nbytes)
    return C, F


class Q4Rows(_Plan):
    """Packed enrol-side rows held in 4 bits (q4_rows makes them)."""

    def __init__(self, codes, scales, q, k, groups):
        self.codes, self.scales, self.q, self.k, self.groups = codes, scales, q, k, groups
        self.device = codes.device
        self._own(codes, scales, q)

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self.codes, self.scales, self.q))

    def values(self):
        """The coordinates that the codes stand for, device fp32 [n, k]."""
        torch = _torch()
        ks = self.codes.shape[1]
        w = self.codes.view(-1, ks, 4, 16, 4)  # block, k-step, coordinates 8 i .. 8 i + 7, row & 15, row >> 4
        shifts = torch.tensor([8 * (j >> 2) + 4 * ((j >> 1) & 1) + 16 * (j & 1) for j in range(8)],
                              dtype=torch.int32, device=w.device)
        c = (w[..., None] >> shifts & 15).float() - 8
        s = (self.scales.view(-1, ks, 1, 16, 4, 1).to(torch.int32) << 16).view(torch.float32)
        v = (c * s).permute(0, 4, 3, 1, 2, 5).reshape(-1, ks * 32)
        g = self.groups
        keep = np.concatenate([np.arange(n) + 64 * b for n, b in zip(g.sizes, _prefix(_ceil(g.sizes, 64)))]
                              or [np.zeros(0)]).astype(np.int64)
        return v[torch.from_numpy(keep).to(v.device)][:, :self.k].contiguous()


def q4_supported(k):
    """Whether the 4-bit operators take rows of k coordinates (1 to 512)."""
    return bool(_lib.load().hypmi_q4_ksteps(int(k)))


def q4_rows(G, k, groups=None):
    """Packed enrol-side rows [g, q, 1] (Plan.prologue; k coordinates) -> Q4Rows.  groups: partitions of the
    gallery (default: one)."""
    torch = require_gpu()
    G, ld = _device_rows(G, _kinds("rows"), "G")
    if groups is None:
        groups = RowGroups([G.shape[0]], device=G.device)
    groups._check(G, "G")
    if groups.order is not None:
        raise ValueError("a gallery needs rows in group order (RowGroups without order)")
    lib = _lib.load()
    ks = lib.hypmi_q4_ksteps(int(k))
    if not ks or G.shape[1] < k + 1:
        raise ValueError("%d coordinates in rows of %d (1 to 512 coordinates, then q)" % (k, G.shape[1]))
    nb = groups._n_tiles[64]
    codes = torch.empty((nb, ks, 64, 4), dtype=torch.int32, device=G.device)
    scales = torch.empty((nb, ks, 16, 4), dtype=torch.int16, device=G.device)
    q = torch.empty((nb, 64), dtype=torch.float32, device=G.device)
    if nb:
        _run(lib.hypmi_q4_rows, G.device, (groups,), G.data_ptr(), ld, int(k), groups._rows[0], groups._rows[2],
             groups.num_groups, nb, codes.data_ptr(), scales.data_ptr(), q.data_ptr())
    return Q4Rows(codes, scales, q, int(k), groups)


def q4_score(gallery, G, pairs, out=None):
    """Scores of packed test-side rows [g, 1, q + c] against a 4-bit gallery, group by group: the flat device
    fp32 result of `pairs` = GroupPairs(test groups, gallery.groups); block e is [tests, gallery rows]."""
    if pairs.cols is not gallery.groups and not np.array_equal(pairs.cols.sizes, gallery.groups.sizes):
        raise ValueError("the columns of pairs are not the groups of the gallery")
    G, ld = _device_rows(G, _kinds("rows"), "G")
    pairs.rows._check(G, "G")
    if gallery.codes.device != pairs.device:
        raise ValueError("the gallery is on %s, the groups on %s" % (gallery.codes.device, pairs.device))
    k, width = gallery.k, G.shape[1]
    if width < k + 2:
        raise ValueError("packed rows of %d elements for a gallery of %d coordinates" % (width, k))
    if G.data_ptr() % 16 or ld % 4 or width < round_up(k, 8):  # not as Plan.prologue leaves them: a padded copy
        ld = round_up(k + 2, 8)
        buf = _torch().zeros((G.shape[0], ld), dtype=G.dtype, device=G.device)
        buf[:, :k + 2] = G[:, :k + 2]
        G = buf
    S = pairs._result(out, G, gallery.codes, gallery.scales, gallery.q)
    if pairs.numel:
        groups = gallery.groups
        _run(_lib.load().hypmi_q4_score, pairs.device, (pairs, pairs.rows, groups, gallery), gallery.codes.data_ptr(),
             gallery.scales.data_ptr(), gallery.q.data_ptr(), gallery.k, G.data_ptr(), ld, pairs.rows._rows[0],
             groups._rows[0], groups._rows[2], pairs._rows[0], pairs._rows[3], pairs._q4_tests, pairs._q4_rows,
             pairs.rows.num_groups, pairs._n_tasks[2], S.data_ptr())
    return S
