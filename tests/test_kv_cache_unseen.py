"""The oracle of the 8-bit cache's attention: a value that is no number reaches the
rows that see its token, and no others."""

import numpy as np
import pytest

from oracle import narrow as N


@pytest.mark.parametrize("causal", [False, True])
def test_oracle_nan_values_reach_the_rows_that_see_them(causal):
    rng = np.random.default_rng(4)
    q, k, v = rng.standard_normal((2, 4, 3, 8)), rng.standard_normal((2, 2, 20, 8)), rng.standard_normal((2, 2, 20, 8))
    scale = np.full((2, 2, 2), 0.5)
    lengths = [20, 2]
    v[0, 1, 18, 5] = v[0, 1, 19, 2] = v[1, 0, 1, 0] = v[0, 0, 3, 7] = v[1, 1, 5, 5] = np.nan
    out = N.kv_cache_attention(q, k, v, scale, scale, lengths, 16, causal, 0.3)
    finite = N.kv_cache_attention(q, k, np.nan_to_num(v), scale, scale, lengths, 16, causal, 0.3)
    for b in range(2):
        for h in range(4):
            for i in range(3):
                end = lengths[b] - 3 + i + 1 if causal else lengths[b]
                reached = np.isnan(v[b, h // 2, : max(end, 0)]).any(0)
                assert np.array_equal(np.isnan(out[b, h, i]), reached)
                assert np.array_equal(out[b, h, i][~reached], finite[b, h, i][~reached])
    assert not causal or not out[1, :, 0].any()
