"""What device plans of transforms are kept by: two chains that compute different things never share a key."""
import numpy as np

from hyperion_amd.transforms import LDA, CentWhiten, LNorm, TransformBank


def test_type_is_part_of_a_transforms_key():
    mu, T = np.arange(3.0), np.eye(3)
    for args in ((), (mu,), (mu, T)):
        assert CentWhiten(*args)._params_key() != LNorm(*args)._params_key()
        assert LNorm(*args)._params_key() == LNorm(*args)._params_key()
    assert CentWhiten(mu, T)._params_key() != LDA(mu, T)._params_key()


def test_a_banks_key_says_which_chain_a_transform_belongs_to():
    def key(*chains):
        return TransformBank(list(chains))._key(3, None)

    L, A = LNorm(), CentWhiten(np.arange(3.0), np.eye(3))
    same = {key([L], [A, L]), key([L, A], [L]), key([L, A, L], []), key([L], [A], [L])}
    assert len(same) == 4
    assert key([L], [A, L]) == key([LNorm()], [CentWhiten(np.arange(3.0), np.eye(3)), L])
