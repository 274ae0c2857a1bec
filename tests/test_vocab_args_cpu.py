"""Arguments of the vocabulary-end operators that are narrowed or laid out before a call, without a GPU."""
import pytest
import torch

import sdmchat_b200 as S
from sdmchat_b200 import vocab as W

BEYOND = [2 ** 32 + 5, -2 ** 32 + 5, 2 ** 31, -2 ** 31 - 1, 2 ** 63 - 1, -2 ** 63]


def test_ids_beyond_32_bits_stay_outside():
    got = W._ids32(torch.tensor(BEYOND + [7, 0, -1]))
    assert got.dtype == torch.int32 and got[-3:].tolist() == [7, 0, -1]
    assert all(v < 0 or v == 2 ** 31 - 1 for v in got[:-3].tolist())
    assert W._ids32(torch.tensor([5, 2 ** 32 - 1], dtype=torch.uint32)).tolist() == [5, 2 ** 31 - 1]
    assert W._ids32(torch.tensor([5, 200], dtype=torch.uint8)).tolist() == [5, 200]


def test_whole_numbers_of_rules_beyond_32_bits():
    wide = torch.tensor([BEYOND[:3], BEYOND[3:]])
    kept = []
    S.LogitRules(history=wide, history_len=torch.tensor([2 ** 32 + 1, -2 ** 32 + 1]), bias_ids=wide,
                 bias_values=torch.zeros(2, 3), mask=torch.full((2, 4), 0xffffffff),
                 mask_row=torch.tensor([2 ** 32, -2 ** 32]))._struct(2, 100, -1, kept)
    history, length, bias, row, mask = kept
    for t in (history, bias):
        assert all(v < 0 or v >= 100 for v in t.flatten().tolist())
    assert length.tolist() == [2 ** 31 - 1, -1] and row.tolist() == [2 ** 31 - 1, -1]
    assert (mask == -1).all()  # words of bits keep their bits


def test_widths_beyond_32_bits_are_refused():
    wide = torch.zeros(1, 1).expand(1, 2 ** 32 + 8)  # one number in memory
    with pytest.raises(ValueError):
        W._rows(wide, "logits")


def test_generate_wants_a_number_per_step():
    """Steps take their numbers from u by index on the device, where an index beyond it could not be refused."""
    m = S.build_onesdm("onesdm_allsdm", 64, dict(d=64, layers=1, mlp_f=176, heads=4, n_sub=8, d_a=8, k=4, chunk=16))
    prompt = torch.zeros(3, 5, dtype=torch.long)
    for shape in ((3, 7), (3, 9), (2, 8), (8,), (3, 8, 1)):
        with torch.no_grad(), pytest.raises(ValueError, match="one number per stream and step"):
            m.generate(prompt, 8, u=torch.rand(shape), temperature=1.0)


def test_lookup_refuses_rows_whose_columns_an_int_does_not_count():
    import ctypes

    from sdmchat_b200 import _lib
    fake = ctypes.c_void_p(0x10000)  # never dereferenced
    for d in (2 ** 30 + 1, 2 ** 31 - 1):
        assert _lib.lib().sdm_embed_scaled(fake, fake, 1, d, 1, 1.0, 1, fake, None, None) == 2
