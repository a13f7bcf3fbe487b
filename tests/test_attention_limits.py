"""Calls of attention over the cache that are refused for their size, before anything runs on a GPU."""
import pytest

T = pytest.importorskip("tetris_amd")
A, B = 4096, 8192  # stand for aligned device addresses: nothing may be read there


@pytest.mark.parametrize("sequences,quanta", [
    (1024, 2 ** 21 - 4),  # 2^31 - 1024 with the three quanta's time that each sequence takes besides
    (512, 2 ** 21),  # (and 8 kv heads) far more
    (2 ** 14, 2 ** 17 - 3),  # 2^31
])
def test_shares_that_would_pass_31_bits(sequences, quanta):
    """All sequences' quanta of 128 tokens are dealt out in shares that are rounded up: 1024 workgroups' shares together may be 1023 quanta more."""
    kv_heads = 8 if sequences == 512 else 1
    assert sequences * kv_heads * (quanta + 3) > 2 ** 31 - 1 - 1024
    c = T.MX4Cache(A, 4, kv_heads, 64, page=16)
    with pytest.raises(T.TetrisError) as e:
        c.attend(A, B, T.BF16, kv_heads, sequences, A, A, 128 * quanta)
    assert e.value.code == T.EUNSUPPORTED


@pytest.mark.parametrize("sequences,heads,most_rows,most_length", [(2 ** 31 - 1, 1024, 40, 2 ** 28), (2 ** 31 - 1, 1, 2 ** 30, 2 ** 28), (2 ** 31 - 1, 1024, 1, 0)])
def test_more_units_than_31_bits_hold(sequences, heads, most_rows, most_length):
    """Units times quanta of the first pass 64 bits; the size that is refused may not be what is left of that."""
    c = T.MX4Cache(A, 4, heads, 32, page=16)
    with pytest.raises(T.TetrisError) as e:
        c.attend(A, B, T.BF16, heads, sequences, A, A, most_length, d_first=A, rows=2 ** 30 // heads, most_rows=most_rows)
    assert e.value.code == T.EUNSUPPORTED
