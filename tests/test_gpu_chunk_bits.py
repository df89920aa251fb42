"""How many bits the attention of several new tokens keeps: its error over a whole output against that of rounding the exact
(64-bit) result to fp16.

Threshold.  The last rounding, to nearest, is off by r = rms(fp16(o) - o), about 2^-12.2 of rms(o): half a step is 2^-12 to 2^-11 of a
value, uniform in it (factor 1 / sqrt 3).  A kernel whose other roundings are those of 32-bit arithmetic and of numbers held in
22 bits (2^-21 of a term, 2^-18 with the sums) adds e below r / 16 in quadrature: rms <= 1.002 r.  One rounding of every weight or of
every query entry to 11 bits adds as much again as r, spread over the terms: 1.2 r and more.  So: rms <= 1.05 r."""
import pytest
import torch

from test_gpu_chunk import _case, _run, _slopes, _want

pytestmark = pytest.mark.gpu


def rounding_ratio(got, want):
    used = ~torch.isnan(want)
    w = want[used]
    rms = lambda x: (x * x).mean().sqrt().item()
    return rms(got[used].double() - w) / rms(w.half().double() - w)


@pytest.mark.parametrize("kr,vr", [([64, 64], [64, 64]), ([128, 16, 80], [112, 64, 32])])
@pytest.mark.parametrize("news,olds", [([1, 5, 8], [900, 300, 0]), ([12], [2000]), ([257], [0]), ([60, 190], [1500, 40]), ([40], [4000])])
def test_error_is_that_of_the_last_rounding(news, olds, kr, vr):
    c = _case(news, olds, kr, vr, D=128, seed=21)
    o, lat, _, _ = _want(c)
    assert rounding_ratio(_run(c, True), o) <= 1.05
    assert rounding_ratio(_run(c, latent=True), lat) <= 1.05


@pytest.mark.parametrize("news", [[6, 2], [150, 20]])
def test_error_with_cap_and_bias(news):
    c = _case(news, [700, 90], [64, 32], [48, 64], seed=22, scale=2.0)
    scores = {"softcap": 20.0, "alibi_slopes": _slopes(2)}
    _, lat, _, _ = _want(c, **scores)
    assert rounding_ratio(_run(c, latent=True, **scores), lat) <= 1.05
