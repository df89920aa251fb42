"""Timing cases of the chunk operators: slot maps, attention of new tokens over the paged latent cache, capped and biased scores.

A serving step adds one or many tokens to every request.  Its slots are found from the request lengths (``maps``), its
tokens attend to everything that is cached before them and to one another (``chunk``), and some models cap the scores, add a
bias that grows with the distance, or mask by window, document or bidirectional prefix (``scores``).

``run`` computes a case in elementary torch operations; with ``own`` set it makes the calls that a program makes of the
library.  ``exact`` states each operator in 64 bits from its definition: keys and values rebuilt from the cache, no absorbed
query, masks as boolean matrices.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"


def listed():
    def maps(name, **kw):
        return {"name": name, "kind": "maps", **kw}

    def attn(name, kind="chunk", **kw):
        c = {"name": name, "kind": kind, "heads": 32, "head_dim": 128, "ragged_ranks": False, "head_major": True, "page": 0,
             "ragged": False, "latent_out": False, "capacity": 0, "graph": False}
        c.update(kw)
        return c

    return [
        # a decode batch's next step in a captured loop: one token each, pages of 16
        maps("maps_decode_64", batch=64, new=1, cached=3001, page=16, ragged=True, rebuild=False, capacity=64, graph=True),
        # prompts admitted together: ragged lengths, pages of 64, some of the buffer unused
        maps("maps_prompts_24", batch=24, new=4096, cached=500, page=64, ragged=True, rebuild=False, capacity=65536, graph=False),
        # five drafted tokens of eight requests verified in one captured step; the buffers hold 64 rows
        attn("chunk_verify_8x5", batch=8, new=5, cached=4091, ragged_ranks=True, page=16, capacity=64, graph=True),
        # a short question behind an image: 117 new tokens over a cached prefix, ranks per head, the reference's layout
        attn("chunk_question_117", batch=1, new=117, cached=2880, ragged_ranks=True, head_major=False, page=64, latent_out=True),
        # a step that mixes decoding requests and pieces of prompts
        attn("chunk_mixed_12", batch=12, new=777, cached=3500, ragged_ranks=True, page=16, ragged=True, latent_out=True),
        # a piece of 512 tokens at the end of a long context
        attn("chunk_512_at_32k", batch=1, new=512, cached=32256, page=64),
        # the largest: a prompt of 8191 tokens in one piece, up to the head outputs
        attn("chunk_prompt_8191", batch=1, new=8191, cached=0),
        # single tokens of a decode batch with a bias by distance (the position signal of the rotary-free form)
        attn("scores_alibi_decode_16", kind="scores", batch=16, new=1, cached=4095, ragged_ranks=True, graph=True,
             latent_out=True, softcap=0.0, alibi=True, window=0, prefix=0, docs=0),
        # capped scores with a sliding window, two prompts
        attn("scores_cap_window_4096", kind="scores", batch=2, new=4096, cached=1000, page=64, ragged=True,
             softcap=50.0, alibi=False, window=1024, prefix=0, docs=0),
        # prompts that begin with 576 image tokens which see one another
        attn("scores_prefix_4x1500", kind="scores", batch=4, new=1500, cached=0, ragged_ranks=True, page=16, ragged=True,
             latent_out=True, softcap=0.0, alibi=False, window=0, prefix=576, docs=0),
        # packed documents of about 700 tokens with a bias by distance
        attn("scores_docs_5000", kind="scores", batch=1, new=5000, cached=0, latent_out=True, softcap=0.0, alibi=True, window=0,
             prefix=0, docs=700),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["maps", "chunk", "chunk", "chunk", "scores", "scores"])
    if kind == "maps":
        batch = _log(rng, 1, 256)
        new = 1 if rng.random() < 0.4 else _log(rng, 1, max(2, min(16384, 65536 // batch)))
        return {"kind": "maps", "batch": batch, "new": new, "cached": rng.choice([0, _log(rng, 1, 8000)]),
                "page": rng.choice([1, 16, 16, 24, 64, 128]), "ragged": rng.random() < 0.6, "rebuild": rng.random() < 0.3,
                "capacity": batch * new + rng.choice([0, 0, 37]), "graph": False}
    shape = rng.choice(["tokens", "drafts", "pieces", "prompt"])
    if shape == "tokens":
        batch, new = _log(rng, 1, 32), 1
    elif shape == "drafts":
        batch, new = _log(rng, 1, 24), rng.randint(2, 16)
    elif shape == "pieces":
        batch, new = _log(rng, 1, 8), _log(rng, 17, 1024)
    else:
        batch, new = 1, _log(rng, 200, 8000)
    # together no more pairs of tokens than the largest listed case, nor more cached tokens than the longest one
    room = min(40000, 100000 // batch, 30_000_000 // (batch * new) - new // 2)
    cached = rng.choice([0, 1, 1]) * (_log(rng, 1, room) if room > 1 else 0)
    heads = rng.choice([32, 32, 40, 8])
    c = {"kind": kind, "batch": batch, "new": new, "cached": cached, "heads": heads, "head_dim": rng.choice([128, 128, 64]),
         "ragged_ranks": rng.random() < 0.6, "head_major": rng.random() < 0.5, "page": rng.choice([0, 1, 16, 64]),
         "ragged": batch > 1 and rng.random() < 0.6, "latent_out": rng.random() < 0.5,
         "capacity": batch * new + rng.choice([0, 0, 19]), "graph": new <= 16 and rng.random() < 0.5}
    if kind == "scores":
        what = rng.choice(["cap", "alibi", "prefix", "docs", "cap_window"])
        c.update(softcap=rng.choice([30.0, 50.0]) if "cap" in what else 0.0, alibi=what in ("alibi", "docs"),
                 window=_log(rng, 16, 4096) if "window" in what else 0, prefix=_log(rng, 2, 1024) if what == "prefix" else 0,
                 docs=_log(rng, 20, 2000) if what == "docs" else 0)
        if c["docs"]:
            c["cached"] = 0
    return c


# ---- lengths and masks: from the case alone ------------------------------------------------------------------------------

_SHARE_NEW = (1.0, 0.0, 0.41, 0.73, 0.0, 0.92, 0.13)
_SHARE_OLD = (0.83, 1.0, 0.52, 0.0, 0.31, 0.67, 0.94, 0.75, 0.11)


def _lengths(case):
    """New and cached tokens of every request; ragged: from single tokens to the full piece."""
    B, new, old = case["batch"], case["new"], case["cached"]
    if not case["ragged"]:
        return [new] * B, [old] * B
    return ([max(1, int(new * _SHARE_NEW[b % 7])) for b in range(B)], [int(old * _SHARE_OLD[b % 9]) for b in range(B)])


def _doc_begin(case, n):
    """First position of the document that each of n packed tokens belongs to; the documents' lengths vary."""
    begin, at, k = np.zeros(n, np.int64), 0, 0
    while at < n:
        size = max(1, int(case["docs"] * (1.0, 0.37, 1.61, 0.82)[k % 4]))
        begin[at:at + size] = at
        at, k = at + size, k + 1
    return begin


def _visible(case):
    """Per request: (first, behind-last) visible position of each new token."""
    out = []
    for n, old in zip(*_lengths(case)):
        pos = old + np.arange(n)
        hi, lo = pos + 1, np.zeros(n, np.int64)
        if case.get("prefix"):
            hi = np.minimum(np.maximum(hi, case["prefix"]), old + n)
        if case.get("window"):
            lo = np.maximum(lo, pos + 1 - case["window"])
        if case.get("docs"):
            lo = np.maximum(lo, _doc_begin(case, n))
        out.append((lo, hi))
    return out


def _ranks(case, shift=0):
    """Per-head ranks: multiples of 16 in [16, 128] with mean 64 over 16 heads."""
    if not case["ragged_ranks"]:
        return [64] * case["heads"]
    steps = [1, 8, 4, 2, 6, 3, 5, 4, 7, 1, 4, 5, 2, 6, 3, 3]
    return [16 * steps[(h + shift) % 16] for h in range(case["heads"])]


def _offsets(ranks):
    return [0] + np.cumsum(ranks).tolist()


def _capacity(case):
    return max(case["capacity"], sum(_lengths(case)[0]))


def work(case):
    news, olds = _lengths(case)
    T = sum(news)
    if case["kind"] == "maps":
        P = case["page"]
        pages = sum(-(-(o + n) // P) - -(-o // P) for n, o in zip(news, olds))
        put = sum(o + n for n, o in zip(news, olds)) if case["rebuild"] else T
        return {"bytes": 4 * (5 * case["batch"] + 2 * _capacity(case) + put + 2 * pages), "flops": 0}
    H, D = case["heads"], case["head_dim"]
    sum_k, sum_v = sum(_ranks(case)), sum(_ranks(case, 5))
    pairs, rows = 0, 0
    for lo, hi in _visible(case):
        pairs += int(np.maximum(hi - lo, 0).sum())
        rows += int(hi.max() - lo.min())
    up = 0 if case["latent_out"] else 1
    moved = 2 * T * H * D + 2 * D * (sum_k + up * sum_v) + rows * (sum_k + sum_v + 4 * H + 4) + 2 * T * (H * D if up else sum_v)
    return {"bytes": moved, "flops": 2 * T * D * (sum_k + up * sum_v) + 2 * pairs * (sum_k + sum_v)}


# ---- inputs: drawn on the GPU from the seed alone -----------------------------------------------------------------------

def _randn(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).half()


def _cache(g, slots, ranks):
    """What a long context has left in a cache: codes of normal latents and one scale per token and head, slot-major."""
    off = _offsets(ranks)
    codes = torch.empty(slots, off[-1], dtype=torch.int8, device=DEV)
    scales = torch.empty(slots, len(ranks), dtype=torch.float16, device=DEV)
    for t in range(0, slots, 16384):
        n = min(16384, slots - t)
        x = _randn(g, n, off[-1])
        for h in range(len(ranks)):
            xh = x[:, off[h]:off[h + 1]]
            s = (xh.abs().amax(1) / 128).clamp_min(1e-4)
            codes[t:t + n, off[h]:off[h + 1]] = torch.round(xh.float() / s.float()[:, None]).clamp(-128, 127).to(torch.int8)
            scales[t:t + n, h] = s
    return codes, scales


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000 + int(seed))
    news, olds = _lengths(case)
    B, T = case["batch"], _capacity(case)
    i32 = dict(dtype=torch.int32, device=DEV)
    width = max(n + o for n, o in zip(news, olds))
    d = {"new": torch.tensor(news, **i32), "old": torch.tensor(olds, **i32),
         "req": torch.randperm(B, generator=g, device=DEV).int()}
    if case["kind"] == "maps":
        P, blocks = case["page"], -(-width // case["page"])
        pool = torch.randperm(2 * B * blocks, generator=g, device=DEV).int()
        d["table"] = pool[:B * blocks].view(B, blocks).clone()            # pages of the cached tokens; the rest is overwritten
        d["free"] = pool[B * blocks:].contiguous()
        d["head"] = torch.randint(0, 1 + B * blocks - sum(-(-(n + o) // P) - -(-o // P) for n, o in zip(news, olds)), (1,),
                                  generator=g, device=DEV).int()
        d["r2t"] = torch.zeros(B, blocks * P, **i32)
        d["slots"] = 2 * B * blocks * P
        return d
    kr, vr = _ranks(case), _ranks(case, 5)
    page = case["page"] or width
    blocks = -(-width // page)
    pool = torch.arange(B * blocks, device=DEV)
    if case["page"]:
        pool = pool[torch.randperm(B * blocks, generator=g, device=DEV)]
    d["r2t"] = (pool.view(B, blocks, 1) * page + torch.arange(page, device=DEV)).view(B, blocks * page).int().contiguous()
    d["slots"] = B * blocks * page
    d["ck"], d["sk"] = _cache(g, d["slots"], kr)
    d["cv"], d["sv"] = _cache(g, d["slots"], vr)
    H, D = case["heads"], case["head_dim"]
    d["q"] = _randn(g, T, H, D)
    d["up_k"] = _randn(g, sum(kr), D, std=0.125)
    d["up_v"] = None if case["latent_out"] else _randn(g, sum(vr), D, std=0.125)
    if case.get("alibi"):
        d["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, dtype=torch.float32, device=DEV) / H)
    if case.get("prefix"):
        d["prefix"] = torch.full((B,), case["prefix"], **i32)
    if case.get("docs"):
        begin = torch.zeros(T, **i32)
        at = 0
        for n in news:
            begin[at:at + n] = torch.from_numpy(_doc_begin(case, n)).to(begin)
            at += n
        d["begin"] = begin
    return d


# ---- what a program has in hand, and one pass ---------------------------------------------------------------------------

def _looped(case, call):
    """The call as a decode loop makes it: captured once over its buffers, or eager."""
    if not case["graph"]:
        return call
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()

    def replay(buffers=call):      # the graph works on the buffers that the call holds
        graph.replay()
        return out
    return replay


def _own_call(case, d):
    from lsvd_b200 import ChunkState, LatentCacheLayout, LatentDecodeAttention, chunk_maps
    if case["kind"] == "maps":
        T = _capacity(case)

        def build():
            m = chunk_maps(d["req"], d["old"], d["new"], d["table"], case["page"], d["r2t"], num_tokens=T, num_slots=d["slots"],
                           free_pages=d["free"], free_head=d["head"], rebuild=case["rebuild"])
            return (m.b_start_loc, m.b_seq_len, m.mem_index, m.position_ids, m.free_head, d["table"], d["r2t"])
        return build
    layout = LatentCacheLayout(_ranks(case), _ranks(case, 5), head_major=case["head_major"])
    caches = d["ck"], d["sk"], d["cv"], d["sv"]
    if case["head_major"]:
        caches = (*layout.to_head_major(d["ck"], d["sk"], "k"), *layout.to_head_major(d["cv"], d["sv"], "v"))
    start = torch.cat([d["new"].new_zeros(1), d["new"].cumsum(0)]).int()
    state = ChunkState(b_req_idx=d["req"], b_seq_len=d["old"] + d["new"], b_start_loc=start, req_to_token=d["r2t"],
                       max_len_in_batch=max(n + o for n, o in zip(*_lengths(case))), max_new_in_batch=max(_lengths(case)[0]))
    attn = LatentDecodeAttention(layout, case["head_dim"], d["up_k"], d["up_v"])
    scores = dict(softcap=case.get("softcap", 0.0), window=case.get("window", 0), alibi_slopes=d.get("slopes"),
                  b_prefix_len=d.get("prefix"), key_begin=d.get("begin"))
    if case["latent_out"]:
        return lambda: (attn.forward_chunk(d["q"], *caches, state, out_latent=d["out"], **scores),)
    return lambda: (attn.forward_chunk(d["q"], *caches, state, out=d["out"], **scores),)


def prepare(case, seed):
    d = _inputs(case, seed)
    if case["kind"] != "maps":     # rows behind the last token stay zero
        d["out"] = torch.zeros(*((_capacity(case), sum(_ranks(case, 5))) if case["latent_out"] else d["q"].shape),
                               dtype=torch.float16, device=DEV)
    return {"case": case, "d": d, "call": _looped(case, _own_call(case, d)) if own else None}


def run(state):
    if own:
        return state["call"]()
    if state["case"]["kind"] == "maps":
        return _plain_maps(state["case"], state["d"])
    return (_plain_attention(state["case"], state["d"]),)


def _plain_maps(case, d):
    B, T, P = case["batch"], _capacity(case), case["page"]
    old, new, row = d["old"].long(), d["new"].long(), d["req"].long()
    seq = old + new
    zero = new.new_zeros(1)
    start = torch.cat([zero, new.cumsum(0)])
    have = (old + P - 1) // P
    need = (seq + P - 1) // P - have
    first = d["head"].long() + torch.cat([zero, need.cumsum(0)])
    # the new pages: page j of request b goes to column have + j of its row
    j = torch.arange(d["table"].shape[1], device=DEV)[None, :]
    fresh = d["free"][(first[:-1, None] + j - have[:, None]).clamp(0, d["free"].numel() - 1)]
    table = d["table"].clone()
    table[row] = torch.where((j >= have[:, None]) & (j < (have + need)[:, None]), fresh, table[row])
    tok = torch.arange(T, device=DEV)
    b = torch.searchsorted(start[1:], tok, right=True).clamp_max(B - 1)
    used = tok < start[-1]
    pos = torch.where(used, old[b] + tok - start[b], torch.zeros_like(tok))
    slot = torch.where(used, table[row[b], pos // P] * P + pos % P, torch.full_like(tok, -1))
    col = torch.arange(d["r2t"].shape[1], device=DEV)[None, :]
    put = (col < seq[:, None]) & (col >= (0 if case["rebuild"] else old[:, None]))
    r2t = d["r2t"].clone()
    r2t[row] = torch.where(put, (table[row][:, col[0] // P] * P + col % P).int(), r2t[row])
    return (start.int(), seq.int(), slot.int(), pos.int(), first[-1:].int(), table, r2t)


def _padded(case, d):
    """Column indexes [heads, 128] of the K and V codes of each head, and which of them exist."""
    got = []
    for ranks in (_ranks(case), _ranks(case, 5)):
        off = torch.tensor(_offsets(ranks), device=DEV)
        j = torch.arange(max(ranks), device=DEV)
        ok = j[None, :] < (off[1:] - off[:-1])[:, None]
        got.append((torch.where(ok, off[:-1, None] + j, torch.zeros_like(j)), ok))
    return got


def _plain_attention(case, d):
    (kc, kok), (vc, vok) = _padded(case, d)
    H, D = case["heads"], case["head_dim"]
    up_k = d["up_k"].float()[kc] * kok[:, :, None]                                # [H, R, D]
    out = d["out"].clone()
    at = 0
    for b, ((lo, hi), n) in enumerate(zip(_visible(case), _lengths(case)[0])):
        lo, hi = torch.from_numpy(lo).to(DEV), torch.from_numpy(hi).to(DEV)
        L = int(_lengths(case)[1][b]) + n
        rows = d["r2t"][d["req"][b].long(), :L].long()
        k = (d["ck"][rows][:, kc].float() * kok).permute(1, 2, 0)                 # [H, R, L]
        v = (d["cv"][rows][:, vc].float() * vok).permute(1, 0, 2)                 # [H, L, R]
        sk, sv = d["sk"][rows].float().t()[:, None, :], d["sv"][rows].float().t()[:, :, None]
        v = v * sv
        t = torch.arange(L, device=DEV)
        step = max(1, min(n, (1 << 27) // (H * L)))
        for i in range(0, n, step):
            e = min(n, i + step)
            qt = d["q"][at + i:at + e].float().permute(1, 0, 2) @ up_k.transpose(1, 2)      # [H, m, R]
            x = (qt @ k) * sk * (1.0 / math.sqrt(D))
            if case.get("softcap"):
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            if case.get("alibi"):
                pos = torch.arange(L - n + i, L - n + e, device=DEV)
                x = x - d["slopes"][:, None, None] * (pos[:, None] - t).abs().float()
            x = torch.where((t >= lo[i:e, None]) & (t < hi[i:e, None]), x, x.new_full((), -math.inf))
            x = torch.exp(x - x.amax(2, keepdim=True))
            o = (x @ v) / x.sum(2, keepdim=True)                                  # [H, m, R]
            if case["latent_out"]:
                out[at + i:at + e] = o.permute(1, 0, 2)[:, vok].half()
            else:
                up_v = d["up_v"].float()[vc] * vok[:, :, None]
                out[at + i:at + e] = (o @ up_v).permute(1, 0, 2).half()
        at += n
    return out


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "maps":
        return _exact_maps(case, {k: (v.cpu().tolist() if isinstance(v, torch.Tensor) else v) for k, v in d.items()})
    H, D = case["heads"], case["head_dim"]
    k_off, v_off = _offsets(_ranks(case)), _offsets(_ranks(case, 5))
    news, olds = _lengths(case)
    out = torch.zeros(_capacity(case), v_off[-1] if case["latent_out"] else H * D, dtype=torch.float64, device=DEV)
    first = 0
    for b in range(case["batch"]):
        n, L = news[b], news[b] + olds[b]
        rows = d["r2t"][int(d["req"][b])][:L].long()
        i, j = torch.arange(n, device=DEV)[:, None] + olds[b], torch.arange(L, device=DEV)[None, :]
        sees = j <= i
        if case.get("prefix"):
            sees = sees | (j < case["prefix"])
        if case.get("window"):
            sees = sees & (i - j < case["window"])
        if case.get("docs"):
            doc = torch.from_numpy(_doc_begin(case, n)).to(DEV)
            sees = sees & (j >= doc[:, None])
        for h in range(H):
            keys = d["sk"][rows, h].double()[:, None] * (d["ck"][rows, k_off[h]:k_off[h + 1]].double() @ d["up_k"][k_off[h]:k_off[h + 1]].double())
            vals = d["sv"][rows, h].double()[:, None] * d["cv"][rows, v_off[h]:v_off[h + 1]].double()
            if not case["latent_out"]:
                vals = vals @ d["up_v"][v_off[h]:v_off[h + 1]].double()
            s = d["q"][first:first + n, h].double() @ keys.t() / math.sqrt(D)
            if case.get("softcap"):
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            if case.get("alibi"):
                s = s - d["slopes"][h].double() * (i - j).abs()
            p = torch.softmax(s.masked_fill(~sees, -math.inf), dim=1)
            cols = slice(v_off[h], v_off[h + 1]) if case["latent_out"] else slice(h * D, (h + 1) * D)
            out[first:first + n, cols] = p @ vals
        first += n
    return (out if case["latent_out"] else out.view(-1, H, D),)


def _exact_maps(case, d):
    P, T = case["page"], _capacity(case)
    start, seq, head = [0], [], d["head"][0]
    slots, positions = [], []
    table, r2t = [list(r) for r in d["table"]], [list(r) for r in d["r2t"]]
    for row, old, new in zip(d["req"], d["old"], d["new"]):
        for block in range(-(-old // P), -(-(old + new) // P)):
            table[row][block] = d["free"][head]
            head += 1
        for pos in range(0 if case["rebuild"] else old, old + new):
            r2t[row][pos] = table[row][pos // P] * P + pos % P
        slots += [table[row][pos // P] * P + pos % P for pos in range(old, old + new)]
        positions += range(old, old + new)
        start.append(start[-1] + new)
        seq.append(old + new)
    tail = T - len(slots)
    return tuple(np.array(x, dtype=np.int32) for x in (start, seq, slots + [-1] * tail, positions + [0] * tail, [head], table, r2t))
