"""Slot maps and attention of several new tokens per request, against plain 64-bit statements of both (oracle/attention.py).

The tolerance of every output is the bound that the oracle derives from the kernels' roundings (chunk_absorb's docstring)."""
import random

import pytest
import torch

import gpu_util as U
from lsvd_b200 import ChunkMaps, ChunkState, LatentCacheLayout, LatentDecodeAttention, chunk_attention_int8_latent_absorb, chunk_maps, synth
from lsvd_b200 import _lib
from oracle import attention as oattn
from oracle import quant

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ---- slot maps ----------------------------------------------------------------------------------------------------------

def _maps_case(B, page, news, olds, seed=0, rows=None, spare=0, free=True, width=None, blocks=None):
    rng = random.Random(seed)
    rows = rows or B + 2
    width = width or max(n + o for n, o in zip(news, olds)) + 5
    blocks = blocks or -(-width // page)
    pages = list(range(2 * rows * blocks + 7))
    rng.shuffle(pages)
    table = [[pages.pop() for _ in range(blocks)] for _ in range(rows)]
    need = sum(-(-(n + o) // page) - -(-o // page) for n, o in zip(news, olds))
    return {"req": rng.sample(range(rows), B), "ready": list(olds), "new": list(news), "table": table, "page": page,
            "r2t": [[-7] * width for _ in range(rows)], "num_tokens": sum(news) + spare, "num_slots": page * (2 * rows * blocks + 7),
            "free": pages[:need + 9] if free else None, "head": 3 if free else 0}


def _run_maps(c, rebuild=False, in_place=False):
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    table, r2t, ready = t(c["table"]), t(c["r2t"]), t(c["ready"])
    status, head, free = t([0]), t([c["head"]]), None if c["free"] is None else t(c["free"])
    out = None
    if in_place:
        new = lambda n: torch.full((n,), -5, dtype=torch.int32, device=DEV)
        out = ChunkMaps(new(len(c["req"]) + 1), ready, new(c["num_tokens"]), new(c["num_tokens"]), head if free is not None else None)
    m = chunk_maps(t(c["req"]), ready, t(c["new"]), table, c["page"], r2t, c["num_tokens"], c["num_slots"], free,
                   head if free is not None else None, rebuild=rebuild, out=out, status_word=status)
    torch.cuda.synchronize()
    return [x if x is None else x.tolist() for x in m], table.tolist(), r2t.tolist(), status.item()


def _check_maps(c, rebuild=False, in_place=False, refused=()):
    got, table, r2t, status = _run_maps(c, rebuild, in_place)
    want_table, want_r2t = [list(r) for r in c["table"]], [list(r) for r in c["r2t"]]
    start, seq, mem, pos, head, bad = oattn.chunk_maps(c["req"], c["ready"], c["new"], want_table, c["page"], want_r2t, c["num_tokens"],
                                                       c["num_slots"], c["free"], c["head"], rebuild)
    assert bad == list(refused)
    assert got[0] == start and got[1] == seq and got[2] == mem and got[3] == pos
    assert got[4] is None if c["free"] is None else got[4] == [head]
    assert table == want_table and r2t == want_r2t
    assert status == (_lib.ERR_BOUNDS if bad else 0)


@pytest.mark.parametrize("B,page,news,olds", [
    (1, 16, [1], [0]), (1, 16, [1], [16]), (3, 1, [1, 4, 2], [0, 3, 9]), (4, 24, [5, 0, 48, 1], [23, 24, 0, 100]),
    (5, 64, [700, 1, 0, 63, 2000], [0, 64, 5, 1, 130]), (2, 1000, [3, 999], [999, 1])])
@pytest.mark.parametrize("rebuild", [False, True])
@pytest.mark.parametrize("free", [False, True])
def test_maps(B, page, news, olds, rebuild, free):
    c = _maps_case(B, page, news, olds, spare=3, free=free)
    _check_maps(c, rebuild)
    _check_maps(c, rebuild, in_place=True)


@pytest.mark.parametrize("B", [64, 257, 1025, 4096])
def test_maps_of_large_batches(B):
    rng = random.Random(B)
    _check_maps(_maps_case(B, 8, [rng.choice([0, 1, 1, 5]) for _ in range(B)], [rng.randrange(0, 30) for _ in range(B)], spare=11), rebuild=B < 2000)


def test_maps_refusals():
    c = _maps_case(6, 16, [2, 3, 4, 5, 6, 7], [0, 10, 20, 30, 40, 50], spare=40)
    _check_maps({**c, "req": c["req"][:2] + [99] + c["req"][3:]}, refused=[2])                    # a row outside the tables
    _check_maps({**c, "req": c["req"][:3] + [c["req"][1]] + c["req"][4:]}, refused=[3])            # the same row twice
    _check_maps({**c, "ready": [0, -1, 20, 30, 40, 50]}, refused=[1])
    _check_maps({**c, "new": [2, -3, 4, 5, 6, 7]}, refused=[1])
    _check_maps({**c, "new": [2, 3, 4000, 5, 6, 7]}, refused=[2, 3, 4, 5])                         # longer than the tables; the rest does not fit
    _check_maps({**c, "num_tokens": 15}, refused=[4, 5])                                           # more tokens than the maps hold
    need = [-(-(n + o) // 16) - -(-o // 16) for n, o in zip(c["new"], c["ready"])]
    assert need == [1, 0, 0, 1, 0, 0]
    _check_maps({**c, "free": c["free"][:c["head"] + 1]}, refused=[3])                             # the free pages run out
    _check_maps({**c, "free": c["free"][:c["head"]]}, refused=[0, 3])
    _check_maps({**c, "head": -1}, refused=[0, 3])
    got, _, r2t, status = _run_maps({**c, "num_slots": 16 * 3})                                    # pages outside the cache
    assert status == _lib.ERR_BOUNDS and all(s < 48 for s in got[2])


def test_maps_same_row_twice_without_new_tokens():
    c = _maps_case(3, 16, [4, 0, 2], [5, 5, 9])
    c["req"][1] = c["req"][0]
    _check_maps(c)


def test_maps_in_a_captured_loop():
    """The replayed step takes pages and advances the lengths by itself."""
    state = ChunkState.paged(rows=3, max_len_in_batch=40, max_tokens=8, max_new_in_batch=3, num_pages=30, page_size=4)
    new = torch.tensor([1, 3, 0], dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        state.begin(new)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        state.begin(new)
    for _ in range(4):
        graph.replay()
    torch.cuda.synchronize()
    assert state.b_seq_len.tolist() == [5, 15, 0] and state.b_start_loc.tolist() == [0, 1, 4, 4]
    assert state.position_ids.tolist() == [4, 12, 13, 14, 0, 0, 0, 0]
    assert state.pages["free_head"].item() == 2 + 4
    r2t = state.req_manager.req_to_token_indexs.cpu()
    slots = torch.cat([r2t[0, :5], r2t[1, :15]])
    assert len(set(slots.tolist())) == 20 and (slots >= 0).all() and (slots < 24).all()
    assert state.mem_index.tolist()[:4] == [r2t[0, 4], r2t[1, 12], r2t[1, 13], r2t[1, 14]]


# ---- attention ----------------------------------------------------------------------------------------------------------

def _case(news, olds, k_ranks, v_ranks, D=64, seed=0, extra=0, scale=1.0):
    lens = [n + o for n, o in zip(news, olds)]
    c = synth.attention_inputs(len(news), len(k_ranks), D, k_ranks, v_ranks, lens, seed, shuffle_slots=True, extra_slots=7)
    c["k_off"], c["v_off"] = U.offsets(k_ranks), U.offsets(v_ranks)
    c["cache_k"], c["scale_k"] = quant.latent_quant_ragged(c["latent_k"], c["k_off"])
    c["cache_v"], c["scale_v"] = quant.latent_quant_ragged(c["latent_v"], c["v_off"])
    g = torch.Generator().manual_seed(seed + 77)
    T = sum(news)
    c["q"] = (torch.randn(T + extra, len(k_ranks), D, generator=g) * scale).half()
    c["start"] = torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=torch.int32)
    c["layout"] = LatentCacheLayout(k_ranks, v_ranks)
    c["T"], c["news"] = T, news
    return c


def _run(c, head_major=False, latent=False, max_new=None, status=None, **scores):
    lay = c["layout"]
    caches = c["cache_k"], c["scale_k"], c["cache_v"], c["scale_v"]
    if head_major:
        caches = (*lay.to_head_major(c["cache_k"], c["scale_k"], "k"), *lay.to_head_major(c["cache_v"], c["scale_v"], "v"))
        lay = lay.as_head_major()
    st = ChunkState(c["b_req_idx"].to(DEV), c["b_seq_len"].to(DEV), c["start"].to(DEV), c["req_to_token"].to(DEV), c["max_len"],
                    max(c["news"]) if max_new is None else max_new)
    dev = {k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in scores.items()}
    T, H, D = c["q"].shape
    out = torch.full((T, H, D) if not latent else (T, lay.sum_v), 77.0, dtype=torch.float16, device=DEV)
    kw = {"out_latent" if latent else "out": out}
    got = chunk_attention_int8_latent_absorb(c["q"].to(DEV), st, H, D, *[t.to(DEV) for t in caches], c["up_k"].to(DEV),
                                             None if latent else c["up_v"].to(DEV), layout=lay, status_word=status, **kw, **dev)
    torch.cuda.synchronize()
    assert got.data_ptr() == out.data_ptr()
    return got.cpu()


def _want(c, **scores):
    names = {"b_prefix_len": "prefix", "alibi_slopes": "slopes"}
    return oattn.chunk_absorb(c["q"], c["cache_k"], c["scale_k"], c["cache_v"], c["scale_v"], c["up_k"], c["up_v"], c["k_off"], c["v_off"],
                              c["req_to_token"], c["b_req_idx"], c["b_seq_len"], c["start"], **{names.get(k, k): v for k, v in scores.items()})


def _close(got, want, tol):
    used = ~torch.isnan(want)
    assert (got[~used] == 77.0).all(), "rows of no request must be left as they were"
    off = (got.double() - want).abs()[used]
    assert torch.isfinite(got[used].float()).all()
    worst = (off / tol[used]).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.2f} times the bound"
    return worst


def _check(c, layouts=(False, True), **scores):
    o, lat, o_tol, lat_tol = _want(c, **scores)
    for hm in layouts:
        _close(_run(c, hm, **scores), o, o_tol)
        _close(_run(c, hm, latent=True, **scores), lat, lat_tol)


RANKS = [([64, 64], [64, 64]), ([16, 128, 48], [128, 16, 80]), ([112, 32], [96, 64])]
LENGTHS = [([1], [0]), ([1], [299]), ([5, 1, 3], [40, 0, 777]), ([16, 2], [16, 128]), ([17], [0]), ([33, 1, 130], [5, 64, 600]),
           ([257], [0]), ([128, 129], [1, 127])]


@pytest.mark.parametrize("kr,vr", RANKS)
@pytest.mark.parametrize("news,olds", LENGTHS)
def test_causal(news, olds, kr, vr):
    _check(_case(news, olds, kr, vr, seed=len(news)))


@pytest.mark.parametrize("D", [8, 24, 72, 128, 256])
@pytest.mark.parametrize("news,olds", [([3, 1], [70, 200]), ([140], [37])])
def test_head_dims(D, news, olds):
    _check(_case(news, olds, [48, 64], [64, 32], D=D), layouts=(False,))


def _slopes(H):
    return 2.0 ** (-8.0 * torch.arange(1, H + 1, dtype=torch.float32) / H)


SCORES = {
    "window": lambda c: {"window": 33},
    "window_1": lambda c: {"window": 1},
    "prefix": lambda c: {"b_prefix_len": torch.tensor([50 + 40 * b for b in range(len(c["news"]))], dtype=torch.int32)},
    "prefix_window": lambda c: {"b_prefix_len": torch.full((len(c["news"]),), 90, dtype=torch.int32), "window": 20},
    "docs": lambda c: {"key_begin": torch.tensor([(i // 13) * 13 for i in range(c["q"].shape[0])], dtype=torch.int32)},
    "full": lambda c: {"causal": False},
    "full_window": lambda c: {"causal": False, "window": 40},
    "cap": lambda c: {"softcap": 3.0},
    "alibi": lambda c: {"alibi_slopes": _slopes(len(c["k_off"]) - 1)},
    "cap_alibi_window": lambda c: {"softcap": 20.0, "alibi_slopes": _slopes(len(c["k_off"]) - 1), "window": 64},
    "alibi_full": lambda c: {"causal": False, "alibi_slopes": _slopes(len(c["k_off"]) - 1)},
    "scale": lambda c: {"sm_scale": 0.3},
}


@pytest.mark.parametrize("name", SCORES)
@pytest.mark.parametrize("news,olds", [([1, 1], [0, 321]), ([7, 12], [90, 3]), ([150, 1, 40], [0, 200, 333])])
def test_scores(name, news, olds):
    c = _case(news, olds, [64, 32], [64, 48], scale=2.0)
    _check(c, layouts=(True,), **SCORES[name](c))


@pytest.mark.parametrize("news", [[4, 2], [60, 150]])
def test_rows_that_see_nothing_are_zero(news):
    c = _case(news, [20, 0], [64, 16], [32, 64])
    begin = torch.zeros(sum(news), dtype=torch.int32)
    begin[1::2] = 100000                                # behind every key
    begin[0] = -5
    _check(c, key_begin=begin)
    assert (_run(c, key_begin=begin)[1::2] == 0).all()


@pytest.mark.parametrize("news", [[3, 5], [40, 140]])
def test_padded_buffers_and_empty_requests(news):
    c = _case([0, news[0], 0, news[1], 0], [30, 11, 0, 90, 7], [64, 48], [64, 16], extra=9)
    _check(c)


@pytest.mark.parametrize("news", [[2, 6], [70, 133]])
def test_unmapped_slots_are_not_seen(news):
    c = _case(news, [60, 35], [64, 48], [64, 16])
    c["req_to_token"][:, 3:40:3] = -1
    c["req_to_token"][:, 32] = -1
    _check(c)


@pytest.mark.parametrize("news", [[2, 6], [70, 133]])
def test_what_masked_keys_hold_touches_nothing(news):
    """Infinities and NaN in the scales of keys that a row does not see (here: everything outside its window)."""
    c = _case(news, [300, 200], [64, 48], [64, 16])
    scores = {"window": 50}
    o, lat, o_tol, lat_tol = _want(c, **scores)
    for b in range(2):
        L, n = int(c["b_seq_len"][b]), news[b]
        rows = c["req_to_token"][int(c["b_req_idx"][b])].long()
        old = rows[:L - n - 50]
        c["scale_k"][old], c["scale_v"][old] = float("inf"), float("nan")
        c["scale_k"][rows[L:]], c["scale_v"][rows[L:]] = float("nan"), float("inf")
    _close(_run(c, **scores), o, o_tol)
    _close(_run(c, True, latent=True, **scores), lat, lat_tol)


@pytest.mark.parametrize("news", [[4], [150]])
def test_a_later_token_that_is_not_finite_leaves_earlier_ones(news):
    """The last token's scales are NaN: only its own row (which sees it) is NaN."""
    c = _case(news, [70], [64, 48], [64, 16])
    o, lat, o_tol, lat_tol = _want(c)
    last = c["req_to_token"][int(c["b_req_idx"][0]), 70 + news[0] - 1].long()
    c["scale_k"][last], c["scale_v"][last] = float("nan"), float("nan")
    got = _run(c)
    assert torch.isnan(got[-1].float()).all()
    got[-1] = 0
    o[-1] = 0
    _close(got, o, o_tol)


@pytest.mark.parametrize("news", [[4], [140]])
def test_extreme_scales_and_queries(news):
    c = _case(news, [200], [64, 128], [64, 128])
    c["scale_v"][:, 0] = 1e-4                        # the smallest scale that the append writes
    c["scale_v"][::7, 1] = 400.0                      # a few huge values among small ones
    c["q"][0] *= 900.0                                # beyond fp16 once absorbed
    c["q"][1] *= 1e-4
    c["q"][2] = 0
    _check(c)


@pytest.mark.parametrize("news", [[2], [130]])
def test_strided_views(news):
    c = _case(news, [50], [64, 32], [48, 64])
    o, lat, o_tol, lat_tol = _want(c)
    T, H, D = c["q"].shape
    lay = c["layout"]
    st = ChunkState(c["b_req_idx"].to(DEV), c["b_seq_len"].to(DEV), c["start"].to(DEV), c["req_to_token"].to(DEV), c["max_len"], max(news))
    wide = lambda t, left, right: torch.nn.functional.pad(t.to(DEV), (left, right))
    q = wide(c["q"].view(T, H * D), 3, 2)[:, 3:-2].unflatten(1, (H, D))         # rows at odd element offsets
    ck, cv = wide(c["cache_k"], 16, 32)[:, 16:-32], wide(c["cache_v"], 32, 16)[:, 32:-16]
    sk, sv = wide(c["scale_k"], 1, 2)[:, 1:-2], wide(c["scale_v"], 3, 0)[:, 3:]
    up_k, up_v = wide(c["up_k"], 1, 0)[:, 1:], wide(c["up_v"], 5, 2)[:, 5:-2]
    out = torch.full((H, T, D + 3), 77.0, dtype=torch.float16, device=DEV)[:, :, 1:-2].transpose(0, 1)
    out_lat = torch.full((T, lay.sum_v + 5), 77.0, dtype=torch.float16, device=DEV)[:, 3:-2]
    chunk_attention_int8_latent_absorb(q, st, H, D, ck, sk, cv, sv, up_k, up_v, layout=lay, out=out, out_latent=out_lat)
    torch.cuda.synchronize()
    _close(out.cpu(), o, o_tol)
    _close(out_lat.cpu(), lat, lat_tol)


def test_bad_bookkeeping_is_reported_and_skipped():
    c = _case([3, 2, 20], [40, 30, 50], [64, 32], [48, 64])
    o, lat, o_tol, lat_tol = _want(c)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    req = c["b_req_idx"].clone()
    c["b_req_idx"][1] = 99                             # an empty request: its rows see nothing
    got = _run(c, latent=True, status=status)
    assert status.item() == _lib.ERR_BOUNDS and (got[3:5] == 0).all()
    lat[3:5] = 0
    _close(got, lat, lat_tol)
    c["b_req_idx"] = req
    o, lat, o_tol, lat_tol = _want(c)
    status.zero_()
    got = _run(c, latent=True, status=status, max_new=3)        # the third request has more: skipped
    assert status.item() == _lib.ERR_BOUNDS
    lat[5:] = float("nan")
    _close(got, lat, lat_tol)
    status.zero_()
    c["req_to_token"][req[0].item(), 7] = c["cache_k"].shape[0] + 5   # a slot outside the cache
    got = _run(c, latent=True, status=status)
    assert status.item() == _lib.ERR_BOUNDS
    c["req_to_token"][req[0].item(), 7] = -1
    _close(got, *[x for x in _want(c)[1::2]])


@pytest.mark.parametrize("news", [[1, 4], [90, 20]])
def test_same_bits_in_both_layouts_and_again(news):
    c = _case(news, [500, 33], [64, 112], [16, 128])
    a = _run(c)
    assert torch.equal(a, _run(c)) and torch.equal(a, _run(c, True))


def test_many_requests_and_long_cache():
    """Splits of the keys, joined by the merge; many requests of one token."""
    c = _case([1] * 40, [(i * 97) % 700 for i in range(40)], [64, 32], [48, 64])
    _check(c)
    c = _case([3], [5000], [64, 32], [48, 64])
    _check(c)
    c = _case([100], [3000], [64, 32], [48, 64])
    _check(c)


def test_steps_together():
    """Maps, append and attention as a server runs them: prompts in pieces, then drafted and single tokens, on a paged cache,
    against the oracle on a cache that was filled by the oracle."""
    kr, vr, D, page = [64, 32], [48, 64], 64, 16
    lay = LatentCacheLayout(kr, vr, head_major=True)
    g = torch.Generator().manual_seed(3)
    state = ChunkState.paged(rows=3, max_len_in_batch=400, max_tokens=300, max_new_in_batch=200, num_pages=80, page_size=page)
    cache = lay.alloc(80 * page, DEV)
    for t in cache:
        t.zero_()
    up_k, up_v = (torch.randn(lay.sum_k, D, generator=g) / 8).half(), (torch.randn(lay.sum_v, D, generator=g) / 8).half()
    attn = LatentDecodeAttention(lay, D, up_k.to(DEV), up_v.to(DEV))
    flat = LatentCacheLayout(kr, vr)
    plain = flat.alloc(80 * page, "cpu")
    for news in ([150, 0, 7], [130, 20, 0], [1, 1, 1], [4, 1, 200], [1, 0, 5]):
        T = sum(news)
        lk, lv = torch.randn(300, lay.sum_k, generator=g).half(), torch.randn(300, lay.sum_v, generator=g).half()
        q = torch.randn(300, 2, D, generator=g).half()
        state.begin(torch.tensor(news, dtype=torch.int32, device=DEV))
        out = attn.forward_chunk(q.to(DEV), *cache, state, latent_k=lk.to(DEV), latent_v=lv.to(DEV), alibi_slopes=_slopes(2).to(DEV))
        torch.cuda.synchronize()
        mem = state.mem_index.cpu()
        assert (mem[T:] == -1).all() and (mem[:T] >= 0).all()
        oattn.cache_append(lk[:T], mem[:T], flat.k_off, plain[0], plain[1])
        oattn.cache_append(lv[:T], mem[:T], flat.v_off, plain[2], plain[3])
        o, _, tol, _ = oattn.chunk_absorb(q, *plain, up_k, up_v, flat.k_off, flat.v_off, state.req_manager.req_to_token_indexs.cpu(),
                                          state.b_req_idx.cpu(), state.b_seq_len.cpu(), state.b_start_loc.cpu(), slopes=_slopes(2))
        off = (out.cpu().double()[:T] - o[:T]).abs()
        assert (off <= tol[:T]).all()


@pytest.mark.parametrize("news", [[2, 1], [140, 30]])
def test_captured_and_replayed_on_another_stream(news):
    c = _case(news, [77, 300], [64, 32], [48, 64])
    o, _, o_tol, _ = _want(c)
    lay = c["layout"]
    st = ChunkState(c["b_req_idx"].to(DEV), c["b_seq_len"].to(DEV), c["start"].to(DEV), c["req_to_token"].to(DEV), c["max_len"], max(news))
    attn = LatentDecodeAttention(lay, 64, c["up_k"].to(DEV), c["up_v"].to(DEV))
    q, caches = c["q"].to(DEV), [c[k].to(DEV) for k in ("cache_k", "scale_k", "cache_v", "scale_v")]
    out = torch.full_like(q, 77.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attn.forward_chunk(q, *caches, st, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            attn.forward_chunk(q, *caches, st, out=out)
        out.fill_(77.0)
        # a larger eager call in between gets a workspace of its own size; the captured step keeps the one it has
        big = _case([60, 60, 60], [900, 900, 900], [64, 32], [48, 64], seed=5)
        bst = ChunkState(big["b_req_idx"].to(DEV), big["b_seq_len"].to(DEV), big["start"].to(DEV), big["req_to_token"].to(DEV), big["max_len"], 60)
        attn.forward_chunk(big["q"].to(DEV), *[big[k].to(DEV) for k in ("cache_k", "scale_k", "cache_v", "scale_v")], bst)
        graph.replay()
        graph.replay()
    side.synchronize()
    _close(out.cpu(), o, o_tol)


def test_two_streams_at_once():
    cases = [_case([9, 30], [400, 77], [64, 32], [48, 64], seed=s) for s in (1, 2)]
    wants = [_want(c) for c in cases]
    dev = [{k: (v.to(DEV) if isinstance(v, torch.Tensor) else v) for k, v in c.items()} for c in cases]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in cases], []
    for c, s in zip(dev, streams):
        st = ChunkState(c["b_req_idx"], c["b_seq_len"], c["start"], c["req_to_token"], c["max_len"], 30)
        with torch.cuda.stream(s):
            outs.append(chunk_attention_int8_latent_absorb(c["q"], st, 2, 64, c["cache_k"], c["scale_k"], c["cache_v"], c["scale_v"],
                                                           c["up_k"], c["up_v"], layout=c["layout"]))
    torch.cuda.synchronize()
    for got, (o, _, tol, _) in zip(outs, wants):
        _close(got.cpu(), o, tol)


@pytest.mark.parametrize("news,olds", [([8], [33]), ([9], [33]), ([8, 9, 16], [500, 0, 64]), ([8] * 5 + [1], [3, 200, 31, 32, 0, 700]),
                                       ([256, 8], [0, 256]), ([16, 17, 15], [300, 70, 0])])
def test_either_side_of_the_two_forms(news, olds):
    """A block of the form for few rows takes eight, a request sixteen."""
    _check(_case(news, olds, [128, 16], [128, 64], seed=8))


@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("news", [[4], [20]])
def test_slots_behind_the_first_four_gigabytes(news, head_major):
    """The case's rows at the end of a cache whose K side has 5 GB: byte offsets pass 32 bits."""
    c = _case(news, [40], [64, 64], [16, 16])
    o, _, o_tol, _ = _want(c)
    n, N = c["cache_k"].shape[0], 40_000_000
    lay = LatentCacheLayout([64, 64], [16, 16], head_major=head_major)
    big = lay.alloc(N, DEV)
    for side, cache, scale, ranks in (("k", big[0], big[1], 64), ("v", big[2], big[3], 16)):
        rows, scales = c["cache_" + side].to(DEV), c["scale_" + side].to(DEV)
        if head_major:
            for h in range(2):
                cache.view(2, N, ranks)[h, N - n:] = rows[:, h * ranks:(h + 1) * ranks]
                scale[h, N - n:] = scales[:, h]
        else:
            cache.view(N, 2 * ranks)[N - n:] = rows
            scale[N - n:] = scales
    r2t = torch.where(c["req_to_token"] >= 0, c["req_to_token"] + (N - n), c["req_to_token"]).to(DEV)
    st = ChunkState(c["b_req_idx"].to(DEV), c["b_seq_len"].to(DEV), c["start"].to(DEV), r2t, c["max_len"], max(news))
    ck, cv = (big[0], big[2]) if head_major else (big[0].view(N, -1), big[2].view(N, -1))
    got = chunk_attention_int8_latent_absorb(c["q"].to(DEV), st, 2, 64, ck, big[1], cv, big[3], c["up_k"].to(DEV), c["up_v"].to(DEV), layout=lay)
    _close(got.cpu(), o, o_tol)


@pytest.mark.parametrize("news", [[3], [30]])
def test_shared_key_and_value_latent(news):
    """One cached latent per head serves K and V: appended once, read as both."""
    ranks, D = [64, 32], 64
    lay, flat = LatentCacheLayout(ranks, shared_kv=True), LatentCacheLayout(ranks, ranks)
    g = torch.Generator().manual_seed(9)
    state = ChunkState.paged(rows=1, max_len_in_batch=100, max_tokens=50, max_new_in_batch=50, num_pages=7, page_size=16)
    cache = lay.alloc(112, DEV)
    plain = flat.alloc(112, "cpu")
    up_k, up_v = (torch.randn(lay.sum_k, D, generator=g) / 8).half(), (torch.randn(lay.sum_k, D, generator=g) / 8).half()
    attn = LatentDecodeAttention(lay, D, up_k.to(DEV), up_v.to(DEV))
    for n in (50, news[0]):
        z, q = torch.randn(n, lay.sum_k, generator=g).half(), torch.randn(n, 2, D, generator=g).half()
        state.begin(torch.tensor([n], dtype=torch.int32, device=DEV))
        out = attn.forward_chunk(q.to(DEV), *cache, state, latent_k=z.to(DEV))
        mem = state.mem_index.cpu()[:n]
        for side in (0, 2):
            oattn.cache_append(z, mem, flat.k_off, plain[side], plain[side + 1])
        o, _, tol, _ = oattn.chunk_absorb(q, *plain, up_k, up_v, flat.k_off, flat.v_off, state.req_manager.req_to_token_indexs.cpu(),
                                          state.b_req_idx.cpu(), state.b_seq_len.cpu(), state.b_start_loc.cpu())
        assert ((out.cpu().double() - o).abs() <= tol).all()


def test_no_tokens():
    c = _case([2], [3], [64, 32], [48, 64])
    lay = c["layout"]
    st = ChunkState(c["b_req_idx"].to(DEV), c["b_seq_len"].to(DEV), torch.zeros(2, dtype=torch.int32, device=DEV), c["req_to_token"].to(DEV), c["max_len"], 0)
    attn = LatentDecodeAttention(lay, 64, c["up_k"].to(DEV), c["up_v"].to(DEV))
    caches = [c[k].to(DEV) for k in ("cache_k", "scale_k", "cache_v", "scale_v")]
    assert attn.forward_chunk(c["q"][:0].to(DEV), *caches, st).shape == (0, 2, 64)
    out = torch.full((2, 2, 64), 77.0, dtype=torch.float16, device=DEV)
    attn.forward_chunk(c["q"].to(DEV), *caches, st, out=out)             # rows, but no request's
    torch.cuda.synchronize()
    assert (out == 77.0).all()
