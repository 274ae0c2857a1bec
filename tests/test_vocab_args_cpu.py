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


def test_outputs_beside_the_logits_in_one_buffer():
    buf = torch.zeros(4, 25)
    for a, b in ((0, 10), (10, 0), (0, 15), (15, 0), (2, 12)):
        assert W._out_rows(buf[:, a:a + 10], buf[:, b:b + 10], "out") == 25
    assert W._out_rows(buf[1:, :10], buf[:3, 10:20], "out") == 25
    assert W._out_rows(buf[:, :10], buf[:, :10], "out") == 25  # the logits themselves
    for a, b in ((0, 9), (9, 0), (1, 0)):
        with pytest.raises(ValueError):
            W._out_rows(buf[:, a:a + 10], buf[:, b:b + 10], "out")
    for out, like in ((buf[1:, :10], buf[:3, :10]), (buf[:, 12:22], buf[:, 3:13]), (buf[1:, :10], buf[:3, 18:])):
        if out.shape == like.shape:
            with pytest.raises(ValueError):
                W._out_rows(out, like, "out")
    flat = torch.zeros(100)
    with pytest.raises(ValueError):  # a row's end and the next one's beginning
        W._out_rows(flat[5:].as_strided((4, 10), (12, 1), 5), flat.as_strided((4, 10), (12, 1), 0), "out")


def test_distillation_refuses_temperatures_whose_reciprocal_or_square_is_infinite():
    import ctypes

    from sdmchat_b200 import _lib
    fake = ctypes.c_void_p(0x10000)  # never dereferenced
    for T in (1e-40, 1e-45, 2e19, 3e38):
        assert _lib.lib().sdm_distill(fake, 100, 3, 100, 0, fake, fake, 4, None, None, None, T, 0.5, 1.0, fake, None, 0,
                                      None) == 1
