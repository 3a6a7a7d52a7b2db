"""The definitions of oracle/qwmx.py against what pins them (CPU)."""
import numpy as np

from oracle import qwmx
from oracle import qworacle as qo


def test_the_token_of_the_rules_is_the_head_fold_s():
    """Infinities, NaN and zeros of both signs: where anything is above -inf, the token that the head's fold names."""
    rng = np.random.default_rng(3)
    pool = np.array([-np.inf, np.nan, -1.0, -0.0, 0.0, 1.0, np.inf], np.float32)
    for top in range(2, len(pool) + 1):
        x = rng.choice(pool[:top], (300, 6)).astype(np.float32)
        l, tokens = qwmx.logits_f32(x)
        assert np.array_equal(l, x, equal_nan=True)
        some = (x > -np.inf).any(axis=1)
        assert np.array_equal(tokens[some], qo.head_argmax(x)[some])
        assert (tokens[~some] == -1).all()
