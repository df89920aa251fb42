"""What a step of several new tokens does with requests that it cannot take: pages that run out, bounds that are passed, rows without
tokens -- through the slot maps, the attention and the layer."""
import pytest
import torch

from lsvd_b200 import ChunkState, LatentCacheLayout, LatentDecodeAttention, LsvdError, _lib, chunk_attention_int8_latent_absorb
from lsvd_b200.chunk import attn_chunk_workspace_bytes
from oracle import attention as oattn
from test_gpu_chunk import _case, _check_maps, _close, _maps_case, _run, _run_maps, _want

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("in_place", [False, True])
def test_a_free_list_without_entries_has_run_out(in_place):
    """It is not a missing one: entries that need a page are refused, the others get their slots, nothing is overwritten."""
    c = _maps_case(4, 16, [2, 3, 20, 5], [0, 10, 20, 32])
    c["free"], c["head"] = [], 0
    _check_maps(c, refused=[0, 2, 3], in_place=in_place)
    _check_maps(c, refused=[0, 2, 3], rebuild=True, in_place=in_place)
    c["head"] = 3                                          # and a head behind its end is no place in it
    _check_maps(c, refused=[0, 2, 3], in_place=in_place)
    got, table, _, status = _run_maps(c)
    assert status == _lib.ERR_BOUNDS and table == c["table"] and got[4] == [3]


class Steps:
    """A paged state over a cache of random latents, with the oracle's copy of it."""

    def __init__(self, rows, num_pages, max_new, page=16, max_len=400, max_tokens=300):
        self.ranks, self.D = ([64, 32], [48, 64]), 64
        self.lay, self.flat = LatentCacheLayout(*self.ranks, head_major=True), LatentCacheLayout(*self.ranks)
        self.g = torch.Generator().manual_seed(31)
        self.state = ChunkState.paged(rows=rows, max_len_in_batch=max_len, max_tokens=max_tokens, max_new_in_batch=max_new,
                                      num_pages=num_pages, page_size=page)
        slots = num_pages * page
        self.cache, self.plain = self.lay.alloc(slots, DEV), self.flat.alloc(slots, "cpu")
        up = lambda n: (torch.randn(n, self.D, generator=self.g) / 8).half()
        self.up = up(self.lay.sum_k), up(self.lay.sum_v)
        self.attn = LatentDecodeAttention(self.lay, self.D, *[u.to(DEV) for u in self.up])

    def step(self, news, **kw):
        """(output with 77 where nothing was written, the oracle's, its bound) of a step; the oracle goes by the state's lengths."""
        T = sum(news)
        make = lambda w: torch.randn(T, w, generator=self.g).half()
        lk, lv, q = make(self.lay.sum_k), make(self.lay.sum_v), make(2 * self.D).view(T, 2, self.D)
        self.state.begin(torch.tensor(news, dtype=torch.int32, device=DEV), **kw)
        out = torch.full((T, 2, self.D), 77.0, dtype=torch.float16, device=DEV)
        self.attn.forward_chunk(q.to(DEV), *self.cache, self.state, latent_k=lk.to(DEV), latent_v=lv.to(DEV), out=out)
        torch.cuda.synchronize()
        st, mem = self.state, self.state.mem_index.cpu()[:T]
        ok = mem >= 0
        oattn.cache_append(lk[ok], mem[ok], self.flat.k_off, self.plain[0], self.plain[1])
        oattn.cache_append(lv[ok], mem[ok], self.flat.v_off, self.plain[2], self.plain[3])
        o, _, tol, _ = oattn.chunk_absorb(q, *self.plain, *self.up, self.flat.k_off, self.flat.v_off,
                                          st.req_manager.req_to_token_indexs.cpu(), st.b_req_idx.cpu(), st.b_seq_len.cpu(), st.b_start_loc.cpu())
        return out.cpu().double(), o, tol


@pytest.mark.parametrize("second", [[2, 8, 1], [2, 40, 1]])
def test_requests_that_find_no_pages_get_zeros(second):
    """The first step takes all five pages of 16; in the second one the second request needs another."""
    s = Steps(rows=3, num_pages=5, max_new=64)
    s.step([20, 9, 30])
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got, want, tol = s.step(second, status_word=status)
    a, e = second[0], second[0] + second[1]
    assert status.item() == _lib.ERR_BOUNDS and s.state.b_seq_len.tolist() == [22, 9, 31]
    assert (s.state.mem_index.cpu()[a:e] == -1).all()
    assert (got[a:e] == 0).all()
    got[a:e], want[a:e] = 0, 0
    assert ((got - want).abs() <= tol).all()


def test_more_new_tokens_than_the_bound_take_no_page():
    """The attention skips a request of more than max_new_in_batch tokens; the maps refuse it before it takes pages or grows."""
    s = Steps(rows=3, num_pages=12, max_new=20)
    s.step([20, 9, 12])
    taken = s.state.pages["free_head"].item()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got, want, tol = s.step([3, 40, 1], status_word=status)
    assert status.item() == _lib.ERR_BOUNDS and s.state.b_seq_len.tolist() == [23, 9, 13]
    assert s.state.pages["free_head"].item() == taken
    assert (s.state.mem_index.cpu()[3:43] == -1).all() and (s.state.req_manager.req_to_token_indexs[1, 9:] == -1).all()
    assert (got[3:43] == 77.0).all()                       # skipped: left as they were
    got[3:43], want[3:43] = 0, 0
    assert ((got - want).abs() <= tol).all()
    got, want, tol = s.step([1, 20, 2])                    # and it goes on from where it was
    assert s.state.b_seq_len.tolist() == [24, 29, 15] and ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("second", [[2, 8, 1], [2, 40, 1], [2, 60, 1]])
def test_the_state_keeps_what_a_step_reports(second):
    """Without a status word of the caller's, eager and replayed: no page left, or more tokens than the bound."""
    s = Steps(rows=3, num_pages=5, max_new=50)
    s.step([20, 9, 30])
    s.state.check()
    s.step(second)
    with pytest.raises(LsvdError):
        s.state.check()
    s.state.check()                                        # once
    new = torch.tensor(second, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            s.state.begin(new)
        graph.replay()
    side.synchronize()
    with pytest.raises(LsvdError):
        s.state.check()


def test_the_state_keeps_what_the_attention_reports():
    """The slot table names a row behind the cache."""
    s = Steps(rows=2, num_pages=8, max_new=30)
    s.step([20, 9])
    s.state.req_manager.req_to_token_indexs[0, 3] = 8 * 16
    s.state.check()
    z = torch.zeros(2, s.lay.sum_k, dtype=torch.float16, device=DEV), torch.zeros(2, s.lay.sum_v, dtype=torch.float16, device=DEV)
    s.state.begin(torch.ones(2, dtype=torch.int32, device=DEV))
    s.attn.forward_chunk(torch.ones(2, 2, s.D, dtype=torch.float16, device=DEV), *s.cache, s.state, latent_k=z[0], latent_v=z[1])
    with pytest.raises(LsvdError):
        s.state.check()


@pytest.mark.parametrize("news", [[3, 5, 4], [30, 50, 40]])
def test_requests_whose_rows_are_not_all_there_are_skipped(news):
    """Rows are a request's last tokens: with some of them missing the others would stand at wrong positions."""
    c = _case(news, [40, 60, 9], [64, 32], [48, 64])
    _, lat, _, tol = _want(c)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    cut = dict(c, q=c["q"][:-2].contiguous())              # the last request lacks two rows
    want = lat[:-2].clone()
    want[news[0] + news[1]:] = float("nan")
    _close(_run(cut, latent=True, status=status), want, tol[:-2])
    assert status.item() == _lib.ERR_BOUNDS
    status.zero_()
    start = c["start"].clone()
    start[0] = -2                                          # in front of the step's rows
    want = lat.clone()
    want[:news[0]] = float("nan")
    _close(_run(dict(c, start=start), latent=True, status=status), want, tol)
    assert status.item() == _lib.ERR_BOUNDS


@pytest.mark.parametrize("news", [[3, 5, 4], [30, 50, 40]])
@pytest.mark.parametrize("causal", [True, False])
def test_requests_with_fewer_tokens_than_rows_see_nothing(news, causal):
    c = _case(news, [40, 60, 9], [64, 32], [48, 64])
    _, lat, _, tol = _want(c, causal=causal)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    lens = c["b_seq_len"].clone()
    lens[1] = news[1] - 1
    lat[news[0]:news[0] + news[1]] = 0
    _close(_run(dict(c, b_seq_len=lens), latent=True, status=status, causal=causal), lat, tol)
    assert status.item() == _lib.ERR_BOUNDS


@pytest.mark.parametrize("captured", [False, True])
def test_one_module_on_two_streams_with_workspaces_of_their_own(captured):
    """Partial results of two steps at once, eager or as graphs that are replayed side by side."""
    cases = [_case([9, 30], [900, 77], [64, 32], [48, 64], seed=s) for s in (1, 2)]
    cases[1]["up_k"], cases[1]["up_v"] = cases[0]["up_k"], cases[0]["up_v"]
    wants = [_want(c) for c in cases]
    attn = LatentDecodeAttention(cases[0]["layout"], 64, cases[0]["up_k"].to(DEV), cases[0]["up_v"].to(DEV))
    runs = []
    for c in cases:
        st = ChunkState(c["b_req_idx"].to(DEV), c["b_seq_len"].to(DEV), c["start"].to(DEV), c["req_to_token"].to(DEV), c["max_len"], 30)
        q, caches = c["q"].to(DEV), [c[k].to(DEV) for k in ("cache_k", "scale_k", "cache_v", "scale_v")]
        out = torch.full_like(q, 77.0)
        ws = torch.empty(attn_chunk_workspace_bytes(st, c["layout"], q.shape[0]), dtype=torch.uint8, device=DEV)
        runs.append((lambda q=q, caches=caches, st=st, out=out, ws=ws: attn.forward_chunk(q, *caches, st, out=out, workspace=ws), out))
    torch.cuda.synchronize()
    streams, calls = [torch.cuda.Stream() for _ in runs], []
    for (call, _), s in zip(runs, streams):
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.stream(s):
                call()
                with torch.cuda.graph(graph, stream=s):
                    call()
            call = graph.replay
        calls.append(call)
    torch.cuda.synchronize()
    for _, out in runs:
        out.fill_(77.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for call, s in zip(calls, streams):
            with torch.cuda.stream(s):
                call()
    torch.cuda.synchronize()
    assert not attn._chunk_workspaces
    for (_, out), (o, _, tol, _) in zip(runs, wants):
        _close(out.cpu(), o, tol)


def test_kept_workspaces_grow_and_stay():
    s = Steps(rows=2, num_pages=40, max_new=200)
    kept = s.attn._chunk_workspaces
    s.step([3, 1])
    first = kept[-1]
    s.step([1, 2])
    assert len(kept) == 1 and kept[0].data_ptr() == first.data_ptr()
    s.step([150, 100])
    assert kept[0].data_ptr() == first.data_ptr() and all(b.numel() >= 2 * a.numel() for a, b in zip(kept, kept[1:]))


def test_tensors_that_are_elsewhere_are_refused():
    """Refused on the host: what the kernels read or write has to be on their device."""
    c = _case([2, 1], [5, 9], [64, 32], [48, 64])
    st = ChunkState(c["b_req_idx"].to(DEV), c["b_seq_len"].to(DEV), c["start"].to(DEV), c["req_to_token"].to(DEV), c["max_len"], 2)
    caches = [c[k].to(DEV) for k in ("cache_k", "scale_k", "cache_v", "scale_v")]

    def call(**kw):
        a = dict(up_k=c["up_k"].to(DEV), up_v=c["up_v"].to(DEV), status_word=None, workspace=None)
        a.update(kw)
        return chunk_attention_int8_latent_absorb(c["q"].to(DEV), st, 2, 64, *caches, layout=c["layout"], **a)

    call()
    word = torch.zeros(1, dtype=torch.int32)
    for bad in (dict(status_word=word), dict(status_word=word.to(DEV).long()), dict(up_k=c["up_k"]), dict(up_v=c["up_v"]),
                dict(workspace=torch.empty(1 << 20, dtype=torch.uint8)), dict(workspace=torch.empty(2 << 20, dtype=torch.uint8, device=DEV)[::2])):
        with pytest.raises(ValueError):
            call(**bad)
    s = Steps(rows=1, num_pages=2, max_new=4)
    with pytest.raises(ValueError):
        s.state.begin(torch.ones(1, dtype=torch.int32, device=DEV), status_word=word)


@pytest.mark.parametrize("news", [[3, 1], [40, 2]])
@pytest.mark.parametrize("causal", [True, False])
def test_bounds_beyond_32_bits_bound_nothing(news, causal):
    c = _case(news, [50, 90], [64, 32], [48, 64])
    want = _run(c, causal=causal)
    for large in (2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 63 - 1):
        assert torch.equal(_run(c, causal=causal, window=large), want)
    s = Steps(rows=2, num_pages=20, max_new=2 ** 32 + 1)
    got, o, tol = s.step(news)
    s.state.check()
    assert ((got - o).abs() <= tol).all()


@pytest.mark.parametrize("swap", [False, True])
@pytest.mark.parametrize("ready,refused", [(5, False), (4, False), (21, True)])
def test_rebuild_of_a_row_that_also_grows(ready, refused, swap):
    """An entry without new tokens is rebuilt beside the one that adds tokens to the same row, unless its length reaches into
    the columns that the new pages go to."""
    c = _maps_case(3, 16, [30, 0, 2], [5, ready, 9])
    c["req"][1] = c["req"][0]
    order = [1, 0, 2] if swap else [0, 1, 2]
    for k in ("req", "ready", "new"):
        c[k] = [c[k][i] for i in order]
    _check_maps(c, rebuild=True, refused=[order.index(1)] if refused else [])
    _check_maps(c)                                         # without a rebuild it reads no column
    if refused:                                            # without a free list no column is written
        c["free"], c["head"] = None, 0
        _check_maps(c, rebuild=True)


@pytest.mark.parametrize("news", [[1, 1, 1], [5, 0, 2]])
def test_a_step_may_have_a_bound_of_its_own(news):
    """The state's bound sizes the grids; a step that is known to bring less may lower it for itself."""
    s = Steps(rows=3, num_pages=30, max_new=200)
    s.step([100, 20, 3])
    s.state.max_new_in_batch = max(news)
    got, want, tol = s.step(news)
    assert ((got - want).abs() <= tol).all()
    s.state.max_new_in_batch = 200
    got, want, tol = s.step([3, 90, 1])
    s.state.check()
    assert ((got - want).abs() <= tol).all()
