"""How many bits the attention of several new tokens keeps: its error over a whole output against that of rounding the exact
(64-bit) result to fp16.

Threshold.  The last rounding, to nearest, is off by r = rms(fp16(o) - o), about 2^-12.2 of rms(o): half a step is 2^-12 to 2^-11 of a
value, uniform in it (factor 1 / sqrt 3).  A kernel whose other roundings are those of 32-bit arithmetic and of numbers held in
22 bits (2^-21 of a term, 2^-17 with the sums over some thousand keys) adds e below r / 16 in quadrature: rms <= 1.002 r.  One rounding of every weight or of
every query entry to 11 bits adds as much again as r, spread over the terms: 1.2 r and more.  So: rms <= 1.05 r."""
import pytest
import torch

from lsvd_b200 import ChunkState, LatentCacheLayout, chunk_attention_int8_latent_absorb
from test_gpu_chunk import _case, _run, _slopes, _want

pytestmark = pytest.mark.gpu
DEV = "cuda"


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


def _ratio_where(got, want, keep):
    rows = torch.where(keep)[0]
    return rounding_ratio(got[rows], want[rows])


@pytest.mark.parametrize("small,large", [(1e-4, 512.0), (1e-4, 65504.0), (0.02, 65504.0)])
@pytest.mark.parametrize("news", [[7, 3], [16, 1], [150, 40]])
@pytest.mark.parametrize("mask", ["window", "docs", "future"])
def test_large_scales_of_masked_keys_cost_no_bits(mask, news, small, large):
    """V scales of the smallest and the largest size: the large ones on keys that a row does not see, in the same tiles as those
    that it sees."""
    c = _case(news, [70, 130], [64, 32], [48, 64], seed=23)
    c["scale_v"][:] = small
    scores, keep = {}, torch.ones(sum(news), dtype=torch.bool)
    if mask == "docs":                       # every row sees its request's keys from 40 on
        scores["key_begin"] = torch.full((sum(news),), 40, dtype=torch.int32)
    if mask == "window":
        scores["window"] = 30
    for b in range(2):
        L, n = int(c["b_seq_len"][b]), news[b]
        rows = c["req_to_token"][int(c["b_req_idx"][b])].long()
        if mask == "docs":
            c["scale_v"][rows[5:40:7]] = large
        elif mask == "window":                # keys that no row sees, and (with many rows) some that only the first rows see
            c["scale_v"][rows[:L - n - 29:5]] = large
            if n > 60:
                c["scale_v"][rows[L - n + 2]] = large
                keep[int(c["start"][b]) + 2:int(c["start"][b]) + 33] = False
        elif n > 1:                           # the last new token, which only its own row sees
            c["scale_v"][rows[L - 1]] = large
            keep[int(c["start"][b]) + n - 1] = False
    o, lat, _, _ = _want(c, **scores)
    got = _run(c, latent=True, **scores)
    assert torch.isfinite(got[keep].float()).all() and _ratio_where(got, lat, keep) <= 1.05
    assert _ratio_where(_run(c, True, **scores), o, keep) <= 1.05


@pytest.mark.parametrize("news", [[5], [140]])
def test_large_scales_of_keys_whose_weight_is_nothing_cost_no_bits(news):
    """The first keys are seen by every row, at distances where the bias leaves less than e^-190 of their weight: 65504 times that is
    nothing to the others, whose scales are 1e-4."""
    c = _case(news, [200], [64, 32], [48, 64], seed=24)
    c["scale_v"][:] = 1e-4
    c["scale_v"][c["req_to_token"][int(c["b_req_idx"][0]), :4].long()] = 65504.0
    scores = {"alibi_slopes": torch.ones(2)}
    _, lat, _, _ = _want(c, **scores)
    assert rounding_ratio(_run(c, latent=True, **scores), lat) <= 1.05


@pytest.mark.parametrize("news", [[5, 1], [140, 33]])
def test_scales_of_zero(news):
    """No V scale, or none of the first keys, has an exponent."""
    c = _case(news, [200, 64], [64, 32], [48, 64], seed=25)
    keep = c["scale_v"].clone()
    c["scale_v"][:] = 0
    assert (_run(c, latent=True) == 0).all()
    for b in range(2):
        rows = c["req_to_token"][int(c["b_req_idx"][b]), 60:int(c["b_seq_len"][b])].long()
        c["scale_v"][rows] = keep[rows]
    _, lat, _, _ = _want(c)
    assert rounding_ratio(_run(c, latent=True), lat) <= 1.05


@pytest.mark.parametrize("cap", [1e-6, 0.5, 30.0, 1e3, 1e4, 1e6, 1e8, 1e30, 3e38])
@pytest.mark.parametrize("news", [[5, 2], [140, 20]])
def test_caps_of_any_size(news, cap):
    """A capped score is off by 2^-19 of itself, never of the cap: one far above the scores changes nothing."""
    c = _case(news, [300, 64], [64, 32], [48, 64], seed=26, scale=6.0)
    _, lat, _, _ = _want(c, softcap=cap)
    assert rounding_ratio(_run(c, latent=True, softcap=cap), lat) <= 1.05
    if cap >= 1e8:
        _, lat, _, _ = _want(c)
        assert rounding_ratio(_run(c, latent=True, softcap=cap), lat) <= 1.05


@pytest.mark.parametrize("news,olds", [([3], [5000]), ([100], [3000]), ([1] * 20, [(i * 97) % 700 + 200 for i in range(20)])])
def test_error_over_splits_of_the_keys(news, olds):
    c = _case(news, olds, [64, 32], [48, 64])
    o, lat, _, _ = _want(c)
    for hm in (False, True):
        assert rounding_ratio(_run(c, hm), o) <= 1.05
        assert rounding_ratio(_run(c, hm, latent=True), lat) <= 1.05


def _exact_long(q, cache_k, scale_k, cache_v, scale_v, up_k, ranks, slots, old, begin=None):
    """Latent result of one request's new tokens in 64 bits, on the GPU (keys rebuilt, dense masks)."""
    T, H, D = q.shape
    out = torch.empty(T, H * ranks, dtype=torch.float64, device=DEV)
    L = old + T
    pos, t = torch.arange(old, L, device=DEV)[:, None], torch.arange(L, device=DEV)[None, :]
    hide = t > pos if begin is None else (t > pos) | (t < begin[:, None])
    for h in range(H):
        c = slice(h * ranks, (h + 1) * ranks)
        keys = scale_k[slots, h].double()[:, None] * (cache_k[slots, c].double() @ up_k[c].double())
        x = (q[:, h].double() @ keys.t() / D ** 0.5).masked_fill_(hide, float("-inf"))
        out[:, c] = torch.softmax(x, 1) @ (scale_v[slots, h].double()[:, None] * cache_v[slots, c].double())
    return out


@pytest.mark.parametrize("heads,new,old,ranks", [(100, 264, 66000, 16), (128, 20, 130000, 16), (32, 40, 8180, 16), (128, 17, 16367, 16),
                                                 (64, 4, 66000, 16), (64, 300, 40000, 112), (74, 300, 8300, 128)])
@pytest.mark.parametrize("begins", [False, True])
def test_long_sums_keep_their_bits(heads, new, old, ranks, begins):
    """Pieces of up to 66000 keys of one block: an accumulator of the tensor cores cuts off what its additions leave, so that its error
    grows with their number (8 for 64 keys), and is folded into fp32 sums every 8192 keys.  The largest scores come late, so that
    references move between the folds; with ``begins`` the rows begin at positions in other tiles, some behind the first fold.

    Threshold: 1024 additions cut off 2^-23 each on average at most, 2^-13 of sums whose terms have one sign (the worst case, here
    nearly so); the last rounding's rms is 2^-12.6 of values like these: sqrt(1 + 2^-0.8) = 1.25.  Without folds 66000 keys come to 4."""
    D = 32
    g = torch.Generator(device=DEV).manual_seed(heads + new)
    L = old + new
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)
    lay = LatentCacheLayout([ranks] * heads)
    codes = lambda: torch.randint(-128, 128, (L, heads * ranks), generator=g, device=DEV, dtype=torch.int8)
    ck, cv = codes(), codes()
    sk = (0.004 + 0.008 * torch.arange(L, device=DEV)[:, None] / L).expand(L, heads).half().contiguous()
    sv = (0.01 + 0.01 * torch.rand(L, heads, generator=g, device=DEV)).half()
    cv = (cv.short() // 2 + 60).clamp(-128, 127).to(torch.int8)      # mostly positive: sums that keep growing
    q, up_k = rand(new, heads, D).half(), (rand(heads * ranks, D) / 8).half()
    slots = torch.randperm(L, generator=g, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    begin = torch.tensor([(i * 977) % (old + 1) for i in range(new)], **i32) if begins else None
    state = ChunkState(torch.zeros(1, **i32), torch.tensor([L], **i32), torch.tensor([0, new], **i32), slots.int()[None], L, new)
    got = chunk_attention_int8_latent_absorb(q, state, heads, D, ck, sk, cv, sv, up_k, layout=lay, key_begin=begin)
    want = _exact_long(q, ck, sk, cv, sv, up_k, ranks, slots, old, begin)
    assert rounding_ratio(got, want) <= 1.25
    up_v = (rand(heads * ranks, D) / 8).half()
    out = chunk_attention_int8_latent_absorb(q, state, heads, D, ck, sk, cv, sv, up_k, up_v, layout=lay, key_begin=begin)
    o = torch.stack([want[:, h * ranks:(h + 1) * ranks] @ up_v[h * ranks:(h + 1) * ranks].double() for h in range(heads)], 1)
    assert rounding_ratio(out, o) <= 1.25
