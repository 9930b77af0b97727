"""The closed-form checks of the paged attention notice the mistakes they are for, planted in the
float64 form (CPU only)."""
import pytest
import torch

from tests._paged import TYPES, attention64
from tests._paged_numbers import beside, closed_form, coded_case, room, sink_case


def rows(args, name):
    """The rows of sequence 0 in order, from the pages."""
    pool = args[name][args["table"][0][args["table"][0] >= 0].long()][:, 0].double()
    return pool.reshape(-1, pool.shape[-1])[:int(args["lens"][0])]


@pytest.mark.parametrize("typ,kv", [("bf16", "bf16"), ("f16", "e4m3")])
def test_closed_form_is_the_definition(typ, kv):
    for args, (ref, lse) in (coded_case([70, 0, 33], 8, 2, 64, 16, typ, kv, "position"),
                             sink_case([70, 1, 33], 8, 2, 64, 16, typ, kv, 9.5)):
        out, l64, _ = attention64(**args)
        assert torch.allclose(out, ref, rtol=1e-12, atol=0)
        assert torch.allclose(l64, lse, rtol=1e-12, atol=0)
        assert not beside(ref.to(TYPES[typ]), ref, room(70, typ, 18)).any()


@pytest.mark.parametrize("n", [130, 5000, 9001])
@pytest.mark.parametrize("code", ["position", "tile"])
def test_lost_and_misplaced_rows_show(n, code):
    args, (ref, _) = coded_case([n], 8, 1, 128, 32, "bf16", "bf16", code)
    k, v = rows(args, "k_pages"), rows(args, "v_pages")

    def seen(v2):
        out, _ = closed_form(args["q"], [k], [v2], args["scale"])
        return beside(out.to(torch.bfloat16), ref, room(n, "bf16")).any()

    assert not seen(v)
    for at in (0, n // 2 // 32 * 32, n // 32 * 32 - 32):
        lost = v.clone()
        lost[at:at + 32] = 0                          # a tile
        assert seen(lost)
        if code == "position":
            lost = v.clone()
            lost[at + 3] = 0                          # a row
            assert seen(lost)
            turned = v.clone()
            turned[at:at + 16] = v[at:at + 16].flip(0)
            assert seen(turned)
        if at + 48 < n:
            swapped = v.clone()
            swapped[at + 16:at + 48] = v[at:at + 32]  # read 16 rows too early
            assert seen(swapped)


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("c", [1.0, 6.0, 9.5])
def test_weights_of_one_term_show(typ, c):
    args, (ref, _) = sink_case([300], 8, 1, 64, 16, typ, typ, c)
    k, v = rows(args, "k_pages"), rows(args, "v_pages")
    one, _ = closed_form(args["q"], [k], [v], c, lambda w: w.to(TYPES[typ]).double())
    far = beside(one.to(TYPES[typ]), ref, room(300, typ, 1.875 * c))
    assert far.any(-1).sum() >= 4                     # of 8 heads


def test_weights_below_2_to_minus_24_lost_show():
    args, (ref, _) = sink_case([300], 8, 1, 64, 16, "f16", "f16", 9.5)
    k, v = rows(args, "k_pages"), rows(args, "v_pages")
    cut, _ = closed_form(args["q"], [k], [v], 9.5, lambda w: (w * 2 ** 24).floor() / 2 ** 24)
    far = beside(cut.half(), ref, room(300, "f16", 18))
    assert far.any(-1).sum() >= 4
