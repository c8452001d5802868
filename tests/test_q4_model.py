"""The plain model of a cache in 4 bits keeps what its definition promises (no GPU)."""
import numpy as np
import pytest

from q4_model import addresses, codes_of


def test_codes_are_nearest():
    """A value (kept within +-2^15, by the definition) is off by half a step s, and at the ends by what rounding m and fifteen s to fp16
    leaves: half a step of fp16 each, 2^-11 of the size or 2^-25 where that is more (fp16's least
    step is 2^-24); s is the rounded one (2^-11 of it more) of an fp32 quotient (2^-22 is enough for that)."""
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((500, 32)) * np.exp(3 * rng.standard_normal((500, 1)))).astype(np.float32)
    c, s, m = codes_of(x)
    x = np.clip(x, -32768, 32768)
    s, m = s.astype(float)[:, None], m.astype(float)[:, None]
    half_m = np.maximum(2.0 ** -11 * np.abs(m), 2.0 ** -25)
    half_s = np.maximum(2.0 ** -11 * s * (1 + 2.0 ** -10), 2.0 ** -25)
    assert (np.abs(x - (m + s * c)) <= s / 2 + half_m + 15 * (half_s + 2.0 ** -22 * s)).all()


@pytest.mark.parametrize("keys", [True, False])
@pytest.mark.parametrize("page,hd", [(16, 32), (32, 96), (64, 256), (256, 128)])
def test_every_byte_of_a_page_is_used_once(page, hd, keys):
    byte, high, scale, low = addresses(page, hd, keys)
    assert sorted((2 * byte + high).ravel().tolist()) == list(range(page * hd))
    ends = np.concatenate([scale[:, ::32].ravel(), low[:, ::32].ravel()])
    assert sorted(ends.tolist()) == list(range(page * hd // 2, page * hd * 5 // 8, 2))
    for j in range(hd // 32):  # all of a group share theirs
        assert (scale[:, 32 * j:32 * j + 32] == scale[:, 32 * j:32 * j + 1]).all()
        assert (low[:, 32 * j:32 * j + 32] == low[:, 32 * j:32 * j + 1]).all()
