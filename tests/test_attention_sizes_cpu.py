"""What an attention call asks for beside its operands: an 8-bit one its own, whatever a 4-bit one needs."""
import pytest

from polar_pack_amd import _native as nat

SIZES = [(2, 128, 64, 100, 128, 128, 16), (8, 128, 64, 200, 64, 64, 64), (2, 64, 16, 50, 3, 12, 8), (2, 256, 64, 500, 2, 2048, 16),
         (1, 192, 32, 40, 1, 1, 6), (4, 128, 64, 300, 2000, 2000, 16)]


@pytest.mark.parametrize("sizes", SIZES)
def test_sizes_of_either_codes(sizes):
    lib = nat.lib()
    for name in ("workspace", "counts"):
        one = getattr(lib, f"pp_kv_attention_codes_{name}_size")
        eight, e4m3, four = (one(c, *sizes) for c in (nat.PP_KV_INT8, nat.PP_KV_E4M3, nat.PP_KV_E2M1))
        assert eight == e4m3 and getattr(lib, f"pp_kv_attention_{name}_size")(*sizes) == max(eight, four)


def test_eight_bits_do_not_pay_for_four():
    """Two workgroups a CU and so twice the parts, of a batch in 4 bits; one in 8."""
    lib = nat.lib()
    for sizes in SIZES[:2]:
        for name in ("workspace", "counts"):
            one = getattr(lib, f"pp_kv_attention_codes_{name}_size")
            assert one(nat.PP_KV_E2M1, *sizes) == 2 * one(nat.PP_KV_INT8, *sizes) > 0


def test_no_sizes():
    lib = nat.lib()
    for name in ("workspace", "counts"):
        assert getattr(lib, f"pp_kv_attention_codes_{name}_size")(nat.PP_KV_E2M1, 2, 64, 16, 3, 2, 0, 4) == 0
