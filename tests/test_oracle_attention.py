"""The attention oracle against closed forms: the e4m3 table and rounding against torch's type, the scale rule, a page filled
token by token against one written at once, rotation as multiplication of complex numbers, softmax rows that see one key or
none."""
import numpy as np
import pytest
import torch

from oracle import attention as ref


def test_e4m3_table_is_torchs():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.E4M3, t, equal_nan=True)


def test_e4m3_rounds_to_the_nearest_even():
    rng = np.random.default_rng(0)
    pos = ref._POSITIVE
    mids = (pos[1:] + pos[:-1]) / 2
    x = np.concatenate([pos, mids, np.nextafter(mids, 0), np.nextafter(mids, 500), rng.uniform(0, 448, 4000),
                        np.exp2(rng.uniform(-14, 8, 4000))]).astype(np.float32)
    x = np.concatenate([x, -x])
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    got = ref.encode_e4m3(x.astype(np.float64))
    assert np.array_equal(ref.E4M3[got], ref.E4M3[want])


@pytest.mark.parametrize("most,want", [(448.0, 1.0), (448.0000001, 2.0), (0.0, 2.0 ** -100), (1e-40, 2.0 ** -100),
                                       (224.0, 0.5), (1.75, 2.0 ** -8), (1.7500001, 2.0 ** -7), (3e38, 2.0 ** 120)])
def test_scale_rule(most, want):
    assert ref.scale_for(most) == want


def test_a_page_filled_token_by_token_is_the_page_written_at_once():
    """Growing by a power of two loses nothing but subnormal codes: with values no more than 2^8 apart there are none."""
    rng = np.random.default_rng(1)
    x = rng.uniform(1, 200, (32, 2, 64)) * rng.choice([-1, 1], (32, 2, 64))
    table = np.array([[1]])
    one, grown = [(np.full((3, 2, 32, 64), 0x7f, np.uint8), np.full((3, 2), np.nan)) for _ in range(2)]
    ref.append(*one, x, [0, 32], [32], table)
    for t in range(32):
        ref.append(*grown, x[t:t + 1], [0, 1], [t + 1], table)
    assert np.array_equal(one[0][1], grown[0][1]) and np.array_equal(one[1][1], grown[1][1])
    assert (one[0][[0, 2]] == 0x7f).all()


def test_rotation_is_a_complex_product():
    rng = np.random.default_rng(2)
    x, pos, freq = rng.standard_normal((5, 3, 10)), np.array([0, 1, 7, 1000, -3]), rng.uniform(0, 1, 4)
    turn = np.exp(1j * pos[:, None] * freq)[:, None, :] * 1.5
    half = ref.rope(x, pos, freq, False, 1.5)
    z = (x[..., :4] + 1j * x[..., 4:8]) * turn
    assert np.allclose(half[..., :4], z.real) and np.allclose(half[..., 4:8], z.imag)
    pairs = ref.rope(x, pos, freq, True, 1.5)
    z = (x[..., 0:8:2] + 1j * x[..., 1:8:2]) * turn
    assert np.allclose(pairs[..., 0:8:2], z.real) and np.allclose(pairs[..., 1:8:2], z.imag)
    assert np.array_equal(half[..., 8:], x[..., 8:]) and np.array_equal(pairs[..., 8:], x[..., 8:])


def test_rows_that_see_one_key_or_none():
    rng = np.random.default_rng(3)
    q, k, v = rng.standard_normal((4, 4, 8)), rng.standard_normal((2, 2, 8)), rng.standard_normal((2, 2, 8))
    out, _ = ref.attend(q, k, v, 0.3)
    assert (out[:2] == 0).all()                       # four rows over two keys: the first two see none
    assert np.allclose(out[2], v[0].repeat(2, 0))     # the third sees the first key alone
    v[1] = np.nan
    assert np.isfinite(ref.attend(q, k, v, 0.3)[0][:3]).all()
