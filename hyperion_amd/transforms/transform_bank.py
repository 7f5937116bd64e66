"""Pre-processing chains by group: every row goes through the chain of its domain, condition or recording."""
import copy

import numpy as np

from .. import engine
from ..fold import fold_chain
from ..hyp_defs import float_cpu
from ..hyp_model import HypModel
from .transform_list import TransformList


class TransformBank(HypModel):
    """One chain of transforms per group of vectors (a TransformList, a transform or a list of them each), e.g. the
    centring, whitening and LDA of several domains: predict(x, ids) puts row i through chains[ids[i]].  In place
    of one TransformList.predict per domain (hyperion/transforms/transform_list.py:41-44) and the gathering of its
    rows; the rows stay where they are, and a step of all chains is one launch.

    The chains have to take the same input dimension, to give the same output dimension and to normalise lengths
    the same number of times; dimensions in between may differ."""

    _cache_defaults = {"_banks": lambda: (None, None)}

    def __init__(self, chains, **kwargs):
        super().__init__(**kwargs)
        if not chains:
            raise ValueError("a TransformBank needs at least one chain")
        self.chains = [list(getattr(c, "transforms", c if isinstance(c, (list, tuple)) else [c])) for c in chains]
        self._banks = (None, None)  # key, maps: replaced together, so that a concurrent call sees both or neither

    def _layers(self, d_in):
        """[(W [E, d_in, d_out], b [E, d_out], dims or None, lnorm)] of the folded chains, float64."""
        folded = [fold_chain([t._step() for t in c], d_in) for c in self.chains]
        if len({len(f[0]) for f in folded}) != 1:
            raise ValueError("the chains normalise lengths a different number of times")
        if len({f[2] for f in folded}) != 1:
            raise ValueError("the chains give vectors of different dimensions")
        steps = [[f[0][i] for f in folded] for i in range(len(folded[0][0]))]  # length-normalised segments
        tails = [f[1] for f in folded]
        layers, E, d = [], len(folded), [d_in] * len(folded)
        for i, step in enumerate(steps + ([tails] if any(A is not None or b is not None for A, b in tails) else [])):
            out = [s[2] for s in step] if i < len(steps) else [folded[0][2]] * E
            W, b = np.zeros((E, max(d), max(out))), np.zeros((E, max(out)))
            for e, s in enumerate(step):
                W[e, :d[e], :out[e]] = np.eye(d[e]) if s[0] is None else s[0]
                if s[1] is not None:
                    b[e, :out[e]] = s[1]
            layers.append((W, b, None if len(set(out)) == 1 else out, i < len(steps)))
            d = out
        return layers

    def _key(self, d_in, device):
        """What the maps laid out on the device are kept by: every chain's transforms, chain by chain."""
        return d_in, device, tuple(tuple(t._params_key() for t in c) for c in self.chains)

    def predict(self, x, ids):
        """x [n, d] (host array, or a device tensor of fp32, fp16 or bf16), ids [n] host integers or a
        RowGroups over the rows of x: [n, d_out], a host array for a host array and a device fp32 tensor for a
        device tensor."""
        torch = engine.require_gpu()
        is_dev = isinstance(x, torch.Tensor)
        if not is_dev or x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
            if not is_dev:
                x = np.asarray(x)
            if x.ndim != 2:
                raise ValueError("expected [num_vectors, dim] input, got shape %s" % (tuple(x.shape),))
            y = engine.upload(x)
        else:
            y = x
        key = self._key(y.shape[1], y.device)
        kept, banks = self._banks
        if kept != key:
            banks = [(engine.AffineBank(W, b, dims=dims, device=y.device), lnorm)
                     for W, b, dims, lnorm in self._layers(y.shape[1])]
            self._banks = key, banks
        if not isinstance(ids, engine.RowGroups):
            if len(ids) != y.shape[0]:
                raise ValueError("%d group ids for %d rows" % (len(ids), y.shape[0]))
            ids = engine.RowGroups.from_ids(ids, len(self.chains), device=y.device)
        for bank, lnorm in banks:
            y = engine.grouped_affine(y, ids, bank, lnorm=lnorm)
        if not banks:  # chains that do nothing
            ids._check(y, "x")
            y = y.to(torch.float32, copy=True)
        return y if is_dev else engine.to_host(y, float_cpu())

    # ---- model files: the transforms of chain e under <name>/<e>/<i>, as a TransformList keeps its own ----------
    def _stored(self):
        prefix = "" if self.name is None else self.name + "/"
        chains = []
        for e, chain in enumerate(self.chains):
            chains.append([copy.copy(t) for t in chain])
            for i, t in enumerate(chains[-1]):
                t.name = "%s%d/%d" % (prefix, e, i)
        return chains

    def save_params(self, f):
        for chain in self._stored():
            for t in chain:
                t.save_params(f)

    @classmethod
    def load_params(cls, f, config):
        chains = config["chains"]
        return cls([TransformList.load_params(f, {"name": None, "transforms": chains[str(e)]}).transforms
                    for e in range(len(chains))], name=config["name"])

    def get_config(self):
        config = super().get_config()
        config["chains"] = {e: {i: t.get_config() for i, t in enumerate(c)} for e, c in enumerate(self._stored())}
        return config
