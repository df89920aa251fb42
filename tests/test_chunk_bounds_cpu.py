"""What the tolerances of the chunk attention's GPU tests are worth: outputs with a planted mistake, computed here in 64 bits, have to
be outside them.  The mistakes are a tile or a key left out, and a rounding to fp16 that the kernels do not make."""
import math

import pytest
import torch

from oracle import attention as oattn, quant
from lsvd_b200 import synth

RATIO = 1.05          # of the GPU tests (test_gpu_chunk_bits.py): error of an output against that of its last rounding


def _rms(x):
    return (x * x).mean().sqrt().item()


def _case(news, olds, k_ranks, v_ranks, D=64, seed=0):
    c = synth.attention_inputs(len(news), len(k_ranks), D, k_ranks, v_ranks, [n + o for n, o in zip(news, olds)], seed, shuffle_slots=True,
                               extra_slots=7)
    off = lambda ranks: [0] + torch.tensor(ranks).cumsum(0).tolist()
    c["k_off"], c["v_off"] = off(k_ranks), off(v_ranks)
    c["cache_k"], c["scale_k"] = quant.latent_quant_ragged(c["latent_k"], c["k_off"])
    c["cache_v"], c["scale_v"] = quant.latent_quant_ragged(c["latent_v"], c["v_off"])
    g = torch.Generator().manual_seed(seed + 77)
    c["q"] = torch.randn(sum(news), len(k_ranks), D, generator=g).half()
    c["start"] = torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=torch.int32)
    return c


def _want(c, table=None):
    return oattn.chunk_absorb(c["q"], c["cache_k"], c["scale_k"], c["cache_v"], c["scale_v"], c["up_k"], c["up_v"], c["k_off"], c["v_off"],
                              c["req_to_token"] if table is None else table, c["b_req_idx"], c["b_seq_len"], c["start"])


LONG = [([3], [5000]), ([100], [3000])]


@pytest.mark.parametrize("news,olds", LONG)
@pytest.mark.parametrize("first,keys", [(1024, 32), (2496, 64), (1791, 1)])
def test_keys_left_out_are_outside_the_bound(news, olds, first, keys):
    """A tile of the stream form, one of the tile form, the last key of a split."""
    c = _case(news, olds, [64, 32], [48, 64])
    o, lat, o_tol, lat_tol = _want(c)
    table = c["req_to_token"].clone()
    table[:, first:first + keys] = -1
    o2, lat2, _, _ = _want(c, table)
    assert ((lat2 - lat).abs() / lat_tol).max() > 2
    if keys > 1:          # a whole tile leaves most entries outside, in the head outputs some
        assert ((lat2 - lat).abs() > lat_tol).double().mean() > 0.5 and ((o2 - o).abs() / o_tol).max() > 2
    # and any of them is far outside the ratio to the last rounding, in both outputs
    for got, want in ((o2, o), (lat2, lat)):
        assert _rms(got.half().double() - want) > 3 * RATIO * _rms(want.half().double() - want)


@pytest.mark.parametrize("news,olds", LONG)
def test_an_output_of_zeros_is_outside_the_bound(news, olds):
    c = _case(news, olds, [64, 64], [64, 64], D=128)
    o, lat, o_tol, lat_tol = _want(c)
    assert (o.abs() <= o_tol).double().mean() < 0.1 and (lat.abs() <= lat_tol).double().mean() < 0.05


def _rounded(c, query=False, weights=False):
    """The latent result in 64 bits with the absorbed query, or the weights times V scales, rounded once to fp16."""
    T, H, D = c["q"].shape
    lat = torch.zeros(T, c["v_off"][-1], dtype=torch.float64)
    half = lambda x, top: (x / top * 256).half().double() / 256 * top         # (entries up to 2^8, as the kernels hold them)
    for b in range(len(c["b_seq_len"])):
        a, e, L = int(c["start"][b]), int(c["start"][b + 1]), int(c["b_seq_len"][b])
        rows = c["req_to_token"][int(c["b_req_idx"][b]), :L].long()
        sees = torch.arange(L)[None, :] <= torch.arange(L - (e - a), L)[:, None]
        for h in range(H):
            ks, vs = slice(c["k_off"][h], c["k_off"][h + 1]), slice(c["v_off"][h], c["v_off"][h + 1])
            qt = c["q"][a:e, h].double() @ c["up_k"][ks].double().t()
            if query:
                qt = half(qt, qt.abs().amax(1, keepdim=True))
            x = (qt @ c["cache_k"][rows, ks].double().t()) * c["scale_k"][rows, h].double() / math.sqrt(D)
            p = torch.softmax(x.masked_fill(~sees, -math.inf), 1)
            w = p * c["scale_v"][rows, h].double()
            if weights:
                w = half(w, w.amax(1, keepdim=True))
            lat[a:e, vs] = w @ c["cache_v"][rows, vs].double()
    return lat


@pytest.mark.parametrize("news,olds", [([1, 5, 8], [900, 300, 0]), ([60, 190], [1500, 40])])
def test_a_rounding_that_the_kernels_do_not_make_is_outside_the_ratio(news, olds):
    c = _case(news, olds, [64, 64], [64, 64], D=128, seed=21)
    _, lat, _, _ = _want(c)
    last = _rms(lat.half().double() - lat)
    assert _rms(_rounded(c) - lat) < 1e-9 * _rms(lat)
    for mistake in (dict(query=True), dict(weights=True)):
        assert _rms(_rounded(c, **mistake).half().double() - lat) > RATIO * last, mistake
