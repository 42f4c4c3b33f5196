"""The bound that the Newton-Schulz GPU tests hold results to: it accepts the model of the kernels'
roundings and tells a result apart that lacks one term of one product, or was made with fewer bits."""
import pytest
import torch

from support.muon_oracle import exact, rel
from support.newton_schulz_model import PRODUCTS, bound, modelled, plain, spectra

SIZES = [(64, 27), (64, 64), (128, 300), (300, 1030), (200, 3000), (512, 640)]


@pytest.mark.parametrize("m,n", SIZES)
def test_a_missing_term_of_any_product_is_found(m, n):
    for name in ("noise", "gradient"):
        x = spectra(m, n, 1)[name]
        want = exact(x)
        most = bound(x, want)
        assert rel(modelled(x), want) <= most and rel(plain(x), want) <= most
        for product in PRODUCTS:
            for term in ((0, 1), (1, 0)):
                assert rel(modelled(x, drop=(product, term)), want) > 2 * most, (name, product, term)


@pytest.mark.parametrize("m,n", [(200, 3000), (256, 2048)])
@pytest.mark.parametrize("name", ["low_rank_0.01", "low_rank_0.001", "column_100000", "falling"])
def test_factors_of_11_bits_are_found_in_a_bf16_result(m, n, name):
    x = spectra(m, n, 1)[name]
    x = (x / x.abs().max()).bfloat16()
    want = exact(x)
    most = bound(x, want, torch.bfloat16)
    assert rel(modelled(x).bfloat16(), want) <= most < rel(modelled(x, wide=False).bfloat16(), want)
