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


def test_a_bank_keeps_its_chains_in_a_model_file(tmp_path):
    """Transforms without names or with the same name in several chains, an empty chain, a chain without parameters."""
    from hyperion_amd.transforms import PCA

    rng = np.random.RandomState(0)
    cw = CentWhiten(rng.randn(4), rng.randn(4, 4), name="cw")
    for name in (None, "bank"):
        bank = TransformBank([[cw, LNorm(), LDA(rng.randn(4), rng.randn(4, 2), name="cw")], [],
                              [CentWhiten(mu=rng.randn(4)), PCA(rng.randn(4), rng.randn(4, 3), pca_dim=3)]], name=name)
        path = str(tmp_path / "bank.h5")
        bank.save(path)
        back = TransformBank.load(path)
        assert back.name == name and [len(c) for c in back.chains] == [3, 0, 2]
        for a, b in zip(sum(bank.chains, []), sum(back.chains, [])):
            assert type(a) is type(b)
            for key in ("mu", "T"):
                x, y = getattr(a, key), getattr(b, key)
                assert (x is None) == (y is None) and (x is None or np.array_equal(x.astype(np.float32), y))
        assert back.chains[2][1].pca_dim == 3 and back.chains[0][2].lda_dim == 2
        assert [t.name for t in bank.chains[0]] == ["cw", None, "cw"]  # saving names nothing anew
        back.save(path)
        again = TransformBank.load(path)
        assert all(np.array_equal(a.T, b.T) for a, b in zip(sum(back.chains, []), sum(again.chains, [])) if a.T is not None)
