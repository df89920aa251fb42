"""Steps of several new tokens per request, without a GPU: what the entry points refuse, and the 64-bit oracle against dense
softmax attention and against a token-by-token walk of the pages."""
import ctypes as C
import random

import pytest
import torch

import lsvd_b200
from lsvd_b200 import _lib, build, synth
from lsvd_b200.attention import LatentCacheLayout
from lsvd_b200.chunk import ChunkMaps, ChunkState, chunk_attention_int8_latent_absorb, chunk_maps
from oracle import attention, quant


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def _maps_args():
    a = _lib.ChunkMapsArgs()
    a.batch, a.page_size, a.num_tokens, a.num_slots = 2, 16, 8, 64
    a.block_table_stride, a.max_blocks, a.table_rows, a.req_to_token_stride, a.max_len = 4, 4, 2, 64, 64
    a.num_free = 4
    for f in ("b_req_idx", "b_ready_cache_len", "b_new_len", "block_table", "req_to_token", "free_pages", "free_head", "free_head_out",
              "b_start_loc", "b_seq_len", "mem_index", "position_ids"):
        setattr(a, f, 4096)
    return a


@pytest.mark.parametrize("change", [
    dict(batch=0), dict(batch=-1), dict(page_size=0), dict(num_tokens=-1), dict(num_slots=0), dict(max_blocks=0), dict(table_rows=0),
    dict(max_len=0), dict(num_free=-1), dict(block_table_stride=3), dict(req_to_token_stride=63), dict(b_req_idx=None),
    dict(b_ready_cache_len=None), dict(b_new_len=None), dict(block_table=None), dict(req_to_token=None), dict(free_head=None),
    dict(free_head_out=None), dict(b_start_loc=None), dict(b_seq_len=None), dict(mem_index=None), dict(position_ids=None),
    dict(mem_index=4098), dict(b_new_len=4097), dict(free_pages=4099)])
def test_maps_refuse_bad_arguments(lib, change):
    a = _maps_args()
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.lsvd_chunk_maps(C.byref(a), None) == _lib.ERR_INVALID_ARG


def test_maps_refuse_larger_batches_than_they_sort(lib):
    a = _maps_args()
    a.batch = _lib.LSVD_MAX_BATCH + 1
    assert lib.lsvd_chunk_maps(C.byref(a), None) == _lib.ERR_UNSUPPORTED
    assert lib.lsvd_chunk_maps(None, None) == _lib.ERR_INVALID_ARG


def _chunk_args(H=2, rank=32):
    a = _lib.AttnChunkArgs()
    a.batch, a.num_heads, a.head_dim, a.max_len_in_batch, a.num_tokens, a.max_new_in_batch, a.num_slots = 2, H, 64, 100, 10, 8, 128
    a.k_off = a.v_off = _lib.i32_array([rank * h for h in range(H + 1)])
    for f in ("q", "cache_k", "scale_k", "cache_v", "scale_v", "up_k", "up_v", "req_to_token", "b_req_idx", "b_seq_len", "b_start_loc",
              "out", "workspace"):
        setattr(a, f, 4096)
    a.q_stride_t, a.q_stride_h, a.out_stride_t, a.out_stride_h = H * 64, 64, H * 64, 64
    a.cache_k_row_stride = a.cache_v_row_stride = H * rank
    a.scale_k_row_stride = a.scale_v_row_stride = H
    a.up_k_row_stride = a.up_v_row_stride = 64
    a.req_to_token_stride, a.req_to_token_rows, a.causal = 100, 2, 1
    a.workspace_bytes = 1 << 40
    return a


@pytest.mark.parametrize("change", [
    dict(batch=0), dict(num_heads=0), dict(num_heads=10 ** 6), dict(head_dim=0), dict(head_dim=63), dict(head_dim=264), dict(num_slots=0),
    dict(max_len_in_batch=-1), dict(num_tokens=-1), dict(max_new_in_batch=-1), dict(k_off=[0, 24, 48]), dict(k_off=[0, 0, 16]),
    dict(v_off=[0, 144, 160]), dict(v_off=[16, 32, 48]), dict(k_off=[0, 32, 16]), dict(q=None), dict(cache_k=None), dict(cache_v=None),
    dict(scale_k=None), dict(scale_v=None), dict(up_k=None), dict(up_v=None), dict(out=None), dict(req_to_token=None),
    dict(b_req_idx=None), dict(b_seq_len=None), dict(b_start_loc=None), dict(cache_layout=7), dict(cache_k=4104), dict(cache_v=4097),
    dict(cache_k_row_stride=63), dict(cache_v_row_stride=48), dict(scale_k_row_stride=1), dict(q=4097), dict(up_k=4097), dict(out=4097),
    dict(b_seq_len=4098), dict(key_begin=4097), dict(b_prefix_len=4099), dict(alibi_slopes=4098), dict(up_k_row_stride=63),
    dict(up_v_row_stride=0), dict(req_to_token_rows=0), dict(req_to_token_stride=99), dict(softcap=float("nan")),
    dict(softcap=float("inf")), dict(softcap=-1.0), dict(window=-1), dict(sm_scale=float("inf")), dict(sm_scale=float("nan"))])
def test_attention_refuses_bad_arguments(lib, change):
    a = _chunk_args()
    for k, v in change.items():
        setattr(a, k, _lib.i32_array(v) if isinstance(v, list) else v)
    assert lib.lsvd_attn_chunk(C.byref(a), None) == _lib.ERR_INVALID_ARG


@pytest.mark.parametrize("change", [dict(max_len_in_batch=(1 << 30) + 1, req_to_token_stride=1 << 31), dict(cache_k_row_stride=1 << 32),
                                    dict(softcap=1e-9), dict(batch=70000)])
def test_attention_refuses_what_it_does_not_reach(lib, change):
    a = _chunk_args()
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.lsvd_attn_chunk(C.byref(a), None) == _lib.ERR_UNSUPPORTED


def test_attention_refuses_a_small_workspace_and_accepts_no_tokens(lib):
    a = _chunk_args()
    need = lib.lsvd_attn_chunk_workspace_bytes(2, 2, 64, 10, 8, 100)
    assert need > 0
    a.workspace_bytes = need - 1
    assert lib.lsvd_attn_chunk(C.byref(a), None) == _lib.ERR_WORKSPACE
    a.workspace_bytes, a.workspace = need, 4096 + 128
    assert lib.lsvd_attn_chunk(C.byref(a), None) == _lib.ERR_WORKSPACE
    a.workspace = None
    assert lib.lsvd_attn_chunk(C.byref(a), None) == _lib.ERR_WORKSPACE
    a.num_tokens = 0
    assert lib.lsvd_attn_chunk(C.byref(a), None) == _lib.OK
    assert lib.lsvd_attn_chunk(None, None) == _lib.ERR_INVALID_ARG
    for bad in ((0, 2, 64, 10, 8, 100), (2, 0, 64, 10, 8, 100), (2, 2, 0, 10, 8, 100), (2, 2, 64, -1, 8, 100), (2, 2, 64, 10, -1, 100)):
        assert lib.lsvd_attn_chunk_workspace_bytes(*bad) == 0


def test_workspace_stays_small_against_the_cache(lib):
    """Partial results are kept for splits only, and a split is hundreds of keys long."""
    for T, new, old in ((8192, 8192, 0), (512, 512, 32768), (64, 1, 4096), (40, 5, 8192), (1, 1, 1 << 20)):
        B = max(1, T // max(new, 1))
        assert lib.lsvd_attn_chunk_workspace_bytes(B, 32, 2048, T, new, new + old) < 1 << 30


def test_cpu_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        chunk_maps(i, i, i, torch.zeros(2, 4, dtype=torch.int32), 16, torch.zeros(2, 64, dtype=torch.int32), 8, 64)
    st = ChunkState(i, i, torch.zeros(3, dtype=torch.int32), torch.zeros(2, 64, dtype=torch.int32), 64, 4)
    z = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        chunk_attention_int8_latent_absorb(z.view(4, 2, 32), st, 2, 32, torch.zeros(64, 32, dtype=torch.int8), z[:, :2],
                                           torch.zeros(64, 32, dtype=torch.int8), z[:, :2], z[:, :32], layout=LatentCacheLayout([16, 16]))
    with pytest.raises(ValueError):
        st.begin(i)                                            # not a paged state


def test_public_names():
    for name in ("ChunkMaps", "ChunkState", "chunk_maps", "chunk_attention_int8_latent_absorb"):
        assert getattr(lsvd_b200, name) is not None
    st = ChunkState.paged(rows=2, max_len_in_batch=33, max_tokens=5, max_new_in_batch=3, num_pages=7, page_size=16, device="cpu")
    assert st.pages["block_table"].shape == (2, 3) and st.pages["num_slots"] == 112 and st.mem_index.tolist() == [-1] * 5


def test_oracle_maps_walk_the_pages():
    rng = random.Random(3)
    for _ in range(20):
        B, page = rng.randrange(1, 6), rng.choice([1, 3, 16])
        olds, news = [rng.randrange(0, 30) for _ in range(B)], [rng.randrange(0, 20) for _ in range(B)]
        width, blocks = 64, -(-64 // page)
        pages = iter(range(1000))
        table = [[-1] * blocks for _ in range(B)]
        for b in range(B):
            for k in range(-(-olds[b] // page)):
                table[b][k] = next(pages)
        free = [next(pages) for _ in range(60)]
        r2t = [[-1] * width for _ in range(B)]
        got = attention.chunk_maps(list(range(B)), olds, news, [list(t) for t in table], page, [list(r) for r in r2t], sum(news) + 2,
                                   1000 * page, free, 0, True)
        taken, at, slots, poss = 0, 0, [], []
        for b in range(B):
            for pos in range(olds[b] + news[b]):
                if pos % page == 0 and table[b][pos // page] < 0:
                    table[b][pos // page] = free[taken]
                    taken += 1
                if pos >= olds[b]:
                    slots.append(table[b][pos // page] * page + pos % page)
                    poss.append(pos)
        assert [list(v) if not isinstance(v, int) else v for v in _fields(got)] == \
            [[sum(news[:b]) for b in range(B + 1)], [o + n for o, n in zip(olds, news)], slots + [-1, -1], poss + [0, 0], taken]


def _fields(got):
    out = []
    for v in got[:5]:
        v = v.tolist() if isinstance(v, torch.Tensor) else v
        out.append(v[0] if isinstance(v, (list, tuple)) and len(out) == 4 else (list(v) if not isinstance(v, int) else v))
    return out


@pytest.mark.parametrize("scores", [dict(), dict(window=5), dict(prefix=[9, 0]), dict(causal=False), dict(causal=False, window=4),
                                    dict(softcap=2.0), dict(alibi=True), dict(docs=True), dict(softcap=1.5, alibi=True, window=7)])
def test_oracle_attention_is_dense_softmax(scores):
    news, olds, H, D, kr, vr = [6, 3], [8, 11], 2, 16, [16, 32], [32, 16]
    c = synth.attention_inputs(2, H, D, kr, vr, [n + o for n, o in zip(news, olds)], 1, shuffle_slots=True, extra_slots=3)
    k_off, v_off = [0, 16, 48], [0, 32, 48]
    ck, sk = quant.latent_quant_ragged(c["latent_k"], k_off)
    cv, sv = quant.latent_quant_ragged(c["latent_v"], v_off)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(sum(news), H, D, generator=g).half()
    start = torch.tensor([0, 6, 9], dtype=torch.int32)
    kw = dict(scores)
    slopes = torch.tensor([0.5, 0.125]) if kw.pop("alibi", False) else None
    begin = torch.tensor([0, 2, 4, 9, 9, 12, 0, 11, 13], dtype=torch.int32) if kw.pop("docs", False) else None
    prefix = torch.tensor(kw.pop("prefix"), dtype=torch.int32) if "prefix" in kw else None
    o, lat, _, _ = attention.chunk_absorb(q, ck, sk, cv, sv, c["up_k"], c["up_v"], k_off, v_off, c["req_to_token"], c["b_req_idx"],
                                          c["b_seq_len"], start, prefix=prefix, key_begin=begin, slopes=slopes, **kw)
    for b in range(2):
        L = news[b] + olds[b]
        rows = c["req_to_token"][int(c["b_req_idx"][b]), :L].long()
        for h in range(H):
            keys = (ck[rows, k_off[h]:k_off[h + 1]].double() * sk[rows, h:h + 1].double()) @ c["up_k"][k_off[h]:k_off[h + 1]].double()
            vals = (cv[rows, v_off[h]:v_off[h + 1]].double() * sv[rows, h:h + 1].double())
            for i in range(news[b]):
                row, pos = int(start[b]) + i, olds[b] + i
                x = keys @ q[row, h].double() / D ** 0.5
                if kw.get("softcap"):
                    x = kw["softcap"] * torch.tanh(x / kw["softcap"])
                t = torch.arange(L)
                if slopes is not None:
                    x = x - slopes[h].double() * (pos - t).abs()
                w = kw.get("window", 0)
                if kw.get("causal", True):
                    sees = (t <= pos) | (t < (int(prefix[b]) if prefix is not None else 0))
                    sees &= (pos - t < w) if w else torch.ones(L, dtype=torch.bool)
                else:
                    sees = ((pos - t).abs() < w) if w else torch.ones(L, dtype=torch.bool)
                if begin is not None:
                    sees &= t >= int(begin[row])
                want = torch.zeros(vals.shape[1], dtype=torch.float64)
                if sees.any():
                    want = torch.softmax(x.masked_fill(~sees, float("-inf")), 0) @ vals
                assert (lat[row, v_off[h]:v_off[h + 1]] - want).abs().max() < 1e-12 * (1 + want.abs().max())
                up = want @ c["up_v"][v_off[h]:v_off[h + 1]].double()
                assert (o[row, h] - up).abs().max() < 1e-12 * (1 + up.abs().max())
