"""Steps of several tokens per request through a layer and a stack of layers (``forward_chunk`` / ``chunk_step``): against the
oracle's stages, against the decode form, in pieces, and as a captured step that takes its own pages."""
import math

import pytest
import torch

from conftest import rel_to_norm
from oracle import attention as oattention, ffn as offn, layer as olayer
from lsvd_b200 import synth
from lsvd_b200.attention import InferState, LatentCacheLayout
from lsvd_b200.chunk import ChunkState
from lsvd_b200.ffn import HybridFFN
from lsvd_b200.layer import LSVDDecoderLayer, make_layer_weights
from lsvd_b200.model import LSVDModel

pytestmark = pytest.mark.gpu

H, D, RQ, HIDDEN, RANK, N_SVD, K = 8, 128, 64, 1024, 128, 384, 12
D_FFN = 12 * 64
KR, VR = synth.ragged_ranks(H, 64, seed=5), synth.ragged_ranks(H, 64, seed=6)


def _weights(n_layers):
    hk = synth.sign_matrix(12, seed=3).float()
    return hk, [(make_layer_weights(HIDDEN, H, D, RQ, KR, VR, seed=10 + 2 * i),
                 synth.ffn_weights(HIDDEN, D_FFN, RANK, N_SVD, seed=11 + 2 * i, had_K=hk, K=K, input_had=False, std=0.05))
                for i in range(n_layers)]


def _layer(head_major=False):
    _, [(lw, fw)] = _weights(1)
    lay = LatentCacheLayout(KR, VR, head_major=head_major)
    to = lambda d: {k: (v.cuda() if isinstance(v, torch.Tensor) else v) for k, v in d.items()}
    return lw, fw, lay, LSVDDecoderLayer(lay, D, RQ, to(lw), HybridFFN(to(fw)))


def _state(max_tokens, max_new, rows=3, max_len=160, page=16):
    return ChunkState.paged(rows=rows, max_len_in_batch=max_len, max_tokens=max_tokens, max_new_in_batch=max_new,
                            num_pages=rows * (-(-max_len // page)), page_size=page)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("head_major", [False, True])
@pytest.mark.parametrize("first,second", [([7, 0, 20], [5, 1, 18]), ([40, 3, 33], [60, 1, 29])])
def test_layer_against_the_oracle(first, second, head_major):
    """Two steps of up to 64 and of more tokens, with a row behind the last one."""
    lw, fw, lay, layer = _layer(head_major)
    st = _state(max_tokens=max(sum(first), sum(second)) + 1, max_new=max(first + second))
    slots = st.pages["num_slots"]
    caches = lay.alloc(slots, "cuda")
    for t in caches:
        t.zero_()
    plain = LatentCacheLayout(KR, VR)
    ref = (torch.zeros(slots, plain.sum_k, dtype=torch.int8), torch.zeros(slots, H, dtype=torch.float16),
           torch.zeros(slots, plain.sum_v, dtype=torch.int8), torch.zeros(slots, H, dtype=torch.float16))
    gen = torch.Generator().manual_seed(3)
    for new in (first, second):
        n = sum(new)
        x = torch.randn(n + 1, HIDDEN, generator=gen).half()
        st.begin(_i32(new))
        stages = {}
        got = layer.forward_chunk(x.cuda(), *caches, st, stages=stages)
        torch.cuda.synchronize()
        # the oracle's stages on the same normalised input (an fp32 mean depends on the order of its additions)
        xn = stages["xn"].cpu()[:n]
        assert rel_to_norm(xn.float(), olayer.rms_norm(x[:n], lw["ln1"], 1e-5).float()) < 1e-3
        lat = olayer.linear_a8w8(xn, lw["W_lat_q"], lw["W_lat_s"])
        assert torch.equal(stages["lat"].cpu()[:n], lat)
        rq = H * RQ
        mem = st.mem_index.cpu()[:n]
        oattention.cache_append(lat[:, rq:rq + plain.sum_k].contiguous(), mem, plain.k_off, ref[0], ref[1])
        oattention.cache_append(lat[:, rq + plain.sum_k:].contiguous(), mem, plain.v_off, ref[2], ref[3])
        ident = torch.zeros(plain.sum_v, RQ, dtype=torch.float16)
        _, o_lat, _, tol = oattention.chunk_absorb(lat[:, :rq].reshape(n, H, RQ), *ref, lw["C"], ident, plain.k_off, plain.v_off,
                                                   st.req_manager.req_to_token_indexs.cpu(), st.b_req_idx.cpu(), st.b_seq_len.cpu(),
                                                   st.b_start_loc.cpu(), sm_scale=1.0 / math.sqrt(D))
        o16 = stages["o_lat"].cpu()
        assert ((o16[:n].double() - o_lat).abs() <= tol).all() and (o16[n:] == 0).all()
        y1 = olayer.linear_a8w8(o16[:n], lw["W_uvo_q"], lw["W_uvo_s"], residual=xn)
        assert torch.equal(stages["y1"].cpu()[:n], y1)
        want = (offn.hybrid_ffn_stages(olayer.rms_norm(y1, lw["ln2"], 1e-6), fw)["out"].float() + y1.float()).half()
        assert rel_to_norm(got.cpu()[:n].float(), want.float()) < 2e-3
    now = [t.cpu() for t in caches]
    if head_major:
        now = [*lay.from_head_major(now[0], now[1], "k"), *lay.from_head_major(now[2], now[3], "v")]
    for a, b in zip(now, ref):
        assert torch.equal(a, b)


def test_one_token_per_request_is_the_decode_step():
    """The two forms of the attention round at different places; everything before it is the same bit for bit."""
    _, _, lay, layer = _layer()
    olds = [70, 1, 33]
    st = _state(max_tokens=sum(olds), max_new=max(olds))
    a = lay.alloc(st.pages["num_slots"], "cuda")
    for t in a:
        t.zero_()
    gen = torch.Generator().manual_seed(4)
    layer.forward_chunk(torch.randn(sum(olds), HIDDEN, generator=gen).half().cuda(), *a, st.begin(_i32(olds)))
    b = [t.clone() for t in a]
    x = torch.randn(3, HIDDEN, generator=gen).half().cuda()
    st.begin(_i32([1, 1, 1]))
    one = ChunkState(st.b_req_idx, st.b_seq_len, st.b_start_loc, st.req_manager.req_to_token_indexs, 160, 1, st.mem_index[:3].contiguous())
    got = layer.forward_chunk(x, *a, one)
    dec = InferState(3, 160, [o + 1 for o in olds], device="cuda", req_to_token=st.req_manager.req_to_token_indexs.cpu())
    want = layer(x, *b, dec)
    for s, t in zip(a, b):
        assert torch.equal(s, t)
    assert rel_to_norm(got.cpu().float(), want.cpu().float()) < 2e-3


def _model(n_layers=2, slots=0):
    hk, ws = _weights(n_layers)
    m = LSVDModel(n_layers, HIDDEN, H, D, D_FFN, RQ, KR, VR, RANK, N_SVD, hk, K, slots, weights=ws)
    for c in m.caches:
        for t in c:
            t.zero_()
    return m


def test_stack_prompt_at_once_and_in_pieces_then_decode():
    lens = [100, 37, 64]
    gen = torch.Generator().manual_seed(5)
    xs = [torch.randn(n, HIDDEN, generator=gen).half().cuda() for n in lens]
    x1 = torch.randn(3, HIDDEN, generator=gen).half().cuda()
    ends = []
    for pieces in (1, 3):
        st = _state(max_tokens=sum(lens), max_new=max(lens))
        m = _model(slots=st.pages["num_slots"])
        done = [0, 0, 0]
        last = [None] * 3
        for k in range(pieces):
            new = [n * (k + 1) // pieces - d for n, d in zip(lens, done)]
            x = torch.cat([xs[b][done[b]:done[b] + new[b]] for b in range(3)])
            pad = torch.zeros(sum(lens) - x.shape[0], HIDDEN, dtype=torch.float16, device="cuda")
            y = m.chunk_step(torch.cat([x, pad]), st.begin(_i32(new)))
            at = 0
            for b in range(3):
                at += new[b]
                last[b] = y[at - 1].clone()
            done = [d + n for d, n in zip(done, new)]
        st.begin(_i32([1, 1, 1]))
        dec = InferState(3, 160, [n + 1 for n in lens], device="cuda", req_to_token=st.req_manager.req_to_token_indexs.cpu())
        ends.append((torch.stack(last).cpu().float(), m.decode_step(x1, dec).cpu().float()))
        assert len({id(layer._chunk_workspaces) for layer in m.layers}) == 1
    # each side is off from the exact stack by what the comparisons with the oracle allow one side (2e-3): twice that
    assert rel_to_norm(ends[0][0], ends[1][0]) < 4e-3 and rel_to_norm(ends[0][1], ends[1][1]) < 4e-3


def test_captured_step_takes_its_pages_and_repeats_the_eager_step():
    """Two captured steps of one model (a wide one and a narrow one), replayed in turn, against eager steps: the same bits."""
    gen = torch.Generator().manual_seed(6)
    wide, narrow = [30, 4, 11], [1, 5, 0]
    xw = [torch.randn(45, HIDDEN, generator=gen).half().cuda() for _ in range(2)]
    xn = [torch.randn(6, HIDDEN, generator=gen).half().cuda() for _ in range(2)]

    def eager():
        st = _state(max_tokens=45, max_new=30)
        m = _model(slots=st.pages["num_slots"])
        outs = []
        for t in range(2):
            outs.append(m.chunk_step(xw[t], st.begin(_i32(wide))).clone())
            sn = ChunkState(st.b_req_idx, st.b_seq_len, st.b_start_loc, st.req_manager.req_to_token_indexs, 160, 30, st.mem_index[:6])
            st.begin(_i32(narrow))
            outs.append(m.chunk_step(xn[t], sn).clone())
        return outs, m, st

    def graphed():
        st = _state(max_tokens=45, max_new=30)
        m = _model(slots=st.pages["num_slots"])
        sn = ChunkState(st.b_req_idx, st.b_seq_len, st.b_start_loc, st.req_manager.req_to_token_indexs, 160, 30, st.mem_index[:6])
        iw, i_n, w, n = xw[0].clone(), xn[0].clone(), _i32(wide), _i32(narrow)
        zero = _i32([0, 0, 0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                # (no token: sizes the workspaces and writes nothing)
            m.chunk_step(i_n, sn)
            m.chunk_step(iw, st.begin(zero))
        torch.cuda.current_stream().wait_stream(side)
        graphs = []
        for x, s, new in ((iw, st, w), (i_n, sn, n)):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                st.begin(new)
                y = m.chunk_step(x, s)
            graphs.append((g, y))
        outs = []
        for t in range(2):
            iw.copy_(xw[t])
            graphs[0][0].replay()
            outs.append(graphs[0][1].clone())
            i_n.copy_(xn[t])
            graphs[1][0].replay()
            outs.append(graphs[1][1].clone())
        torch.cuda.synchronize()
        return outs, m, st

    a, ma, sa = eager()
    b, mb, sb = graphed()
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    assert torch.equal(sa.b_seq_len, sb.b_seq_len) and torch.equal(sa.req_manager.req_to_token_indexs, sb.req_manager.req_to_token_indexs)
    for ca, cb in zip(ma.caches, mb.caches):
        for s, t in zip(ca, cb):
            assert torch.equal(s, t)
