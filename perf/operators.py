"""Workloads of the operators on a KV cache whose slots are not positions.

Four operators that meet in one cache (fp16 keys and values, fp32
activations): rotary positions with a store into given slots, attention of a
tree of drafted tokens over the cache, the choice of the positions that an
eviction keeps, and the move of chosen rows. `own` says which side `run`
calls: the plain form in torch, or this repository's library.
"""
import math
import random

import numpy as np
import torch

own = False
DEV = "cuda"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _attend(name, **kw):
    c = dict(name=name, op="attend", seqs=1, tokens=1, ctx=512, ragged=False, tree=True, nqh=32, nkh=8, hd=128,
             head_major=False, cap=0.0, window=0, slopes=False, slots="plain", weights=False)
    c.update(kw)
    return c


def _rope(name, **kw):
    c = dict(name=name, op="rope", tokens=1, seqs=1, ctx=4096, nqh=32, nkh=8, hd=128, rot=128, axes=1,
             interleaved=False, halves=False, factors=False, head_major=False, far=0)
    c.update(kw)
    return c


def _select(name, **kw):
    c = dict(name=name, op="select", layers=1, seqs=1, heads=8, n=4096, keep=1024, first=4, recent=128, ragged=False)
    c.update(kw)
    return c


def _gather(name, **kw):
    c = dict(name=name, op="gather", layers=32, seqs=1, heads=8, hd=128, ctx=8192, n=2048, accept=False,
             head_major=False)
    c.update(kw)
    return c


def listed():
    return [
        # one new token of one sequence early in a chat: only latency counts (8B shape: 32/8 heads of 128)
        _attend("attend_one_token", ctx=499),
        # a tree of 16 drafts verified in one pass at the 8B shape's context of 4096
        _attend("attend_tree16_ctx4096", tokens=16, ctx=4080),
        # a wide tree (odd size) at the 70B shape (64/8 heads of 128, context 8192), head-major cache
        _attend("attend_tree63_ctx8192", tokens=63, ctx=8129, nqh=64, head_major=True),
        # 16 sequences of different lengths with short chains of drafts, heads of 256, capped scores, a sliding window
        _attend("attend_ragged_window", seqs=16, tokens=5, ctx=8001, ragged=True, tree=False, nqh=16, hd=256, cap=50.0,
                window=4096),
        # one rank's KV head of the 70B shape over 8 GPUs on a very long context, linear distance bias
        _attend("attend_long_bias", tokens=7, ctx=131065, nqh=8, nkh=1, head_major=True, slopes=True),
        # the last 32 prompt tokens as the observation window of an eviction: four left-padded prompts, weights out
        _attend("attend_weights", seqs=4, tokens=32, ctx=4064, tree=False, slots="padded", weights=True),
        # a decode batch of 8: one token each, new positions of a cache that was cut before (slot < position)
        _rope("rope_batch8", tokens=8, seqs=8, far=100000),
        # a prompt with images: three position axes, half-split pairs, 70B heads
        _rope("rope_images", tokens=4093, nqh=64, axes=3, halves=True, interleaved=True),
        # one layer's choice in the middle of decoding: 8 lists
        _select("select_one_layer"),
        # all 32 layers of four prompts at once, different lengths
        _select("select_prompts", layers=32, seqs=4, n=16384, keep=2047, recent=256, ragged=True),
        # the accepted branch of a draft tree moves behind the context: 8 sequences, all layers, a few rows each
        _gather("gather_accept", seqs=8, ctx=512, n=5, accept=True),
        # an 8192-token prompt's cache cut to 2048 positions per head, all layers, into the smaller decode cache
        _gather("gather_evict"),
    ]


#: The dearest listed cases: a drawn one stays under these.
_MOST_FLOPS = 17e9
_MOST_BYTES = 500e6


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.4)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "rope", "select", "gather"])
    heads = rng.choice([1, 2, 4, 8])
    hd = rng.choice([32, 64, 64, 80, 96, 112, 128, 128, 128, 256])
    if op == "attend":
        while True:
            slots = rng.choice(["plain", "plain", "padded", "evicted"])
            c = _attend("", seqs=_log(rng, 1, 32), tokens=_log(rng, 1, 200), ctx=_log(rng, 3, 100000),
                        ragged=rng.random() < 0.5, tree=rng.random() < 0.6, nqh=heads * rng.choice([1, 2, 3, 4, 5, 7, 8]),
                        nkh=heads, hd=hd, head_major=rng.random() < 0.5, cap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                        window=rng.choice([0, 0, 0, 100, 1024]), slopes=rng.random() < 0.3, slots=slots,
                        weights=rng.random() < 0.25)
            del c["name"]
            w = work(c)
            # the plain form holds all scores at once: bounded too
            if (w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES and
                    c["seqs"] * c["nqh"] * c["tokens"] * (c["ctx"] + c["tokens"]) <= 1.5e8):
                return c
    if op == "rope":
        axes = rng.choice([1, 1, 2, 3, 4])
        rot = hd if rng.random() < 0.7 else hd // 2
        c = _rope("", seqs=_log(rng, 1, 16), nqh=heads * rng.choice([1, 2, 4, 5, 8]), nkh=heads, hd=hd, rot=rot, axes=axes,
                  interleaved=axes > 1 and rng.random() < 0.5, halves=rng.random() < 0.5, factors=rng.random() < 0.3,
                  head_major=rng.random() < 0.5, far=rng.choice([0, 1000, 100000, 1000000]))
        c["tokens"] = _log(rng, 1, 4096)
        c["ctx"] = c["tokens"] + rng.randrange(1, 4000)
        del c["name"]
        return c
    if op == "select":
        c = _select("", layers=rng.choice([1, 2, 8, 32]), seqs=_log(rng, 1, 4), heads=heads, n=_log(rng, 17, 16384),
                    ragged=rng.random() < 0.5, first=rng.choice([0, 1, 4, 16]))
        c["keep"] = max(1, int(c["n"] * rng.uniform(0.05, 1.1)))
        c["first"] = min(c["first"], c["keep"])
        c["recent"] = rng.randrange(0, c["keep"] - c["first"] + 1)
        del c["name"]
        return c
    while True:
        c = _gather("", layers=rng.choice([1, 4, 32]), seqs=_log(rng, 1, 8), heads=heads, hd=hd, accept=rng.random() < 0.5,
                    head_major=rng.random() < 0.5)
        c["ctx"] = _log(rng, 64, 8192)
        c["n"] = rng.randrange(2, 12) if c["accept"] else max(1, int(c["ctx"] * rng.uniform(0.05, 1.0)))
        del c["name"]
        if c["layers"] * c["seqs"] * heads * c["ctx"] * hd <= 32 * 8 * 8192 * 128 and work(c)["bytes"] <= _MOST_BYTES:
            return c


def _lengths(c):
    """(context positions, new tokens) of every sequence of an attend case."""
    if not c["ragged"]:
        return [c["ctx"]] * c["seqs"], [c["tokens"]] * c["seqs"]
    r = random.Random(c["ctx"] * 131 + c["seqs"])
    return ([max(0, int(c["ctx"] * r.uniform(0.1, 1.0))) if i else c["ctx"] for i in range(c["seqs"])],
            [r.randint(1, c["tokens"]) if i else c["tokens"] for i in range(c["seqs"])])


def _counts(c):
    """Scored positions of every sequence of a select case."""
    if not c["ragged"]:
        return [c["n"]] * c["seqs"]
    r = random.Random(c["n"] * 17 + c["seqs"])
    return [max(1, int(c["n"] * r.uniform(0.1, 1.0))) if i else c["n"] for i in range(c["seqs"])]


def work(case):
    c = case
    if c["op"] == "attend":
        nc, nt = _lengths(c)
        group = c["nqh"] // c["nkh"]
        keys = pairs = 0
        for n, t in zip(nc, nt):
            seen = min(n, c["window"] + t) if c["window"] and c["slots"] == "plain" else n
            keys += seen + t
            pairs += t * (min(n, c["window"]) if c["window"] else n) + t * (t + 1) // 2
        b = keys * c["nkh"] * c["hd"] * 2 * 2 + 2 * sum(nt) * c["nqh"] * c["hd"] * 4
        b += sum(nt) * ((c["tokens"] + 31) // 32) * 4 if c["tree"] else 0
        b += keys * 4 * (c["nkh"] if c["slots"] == "evicted" else 1) if c["slots"] != "plain" else 0
        b += 2 * keys * c["nkh"] * 4 if c["weights"] else 0
        return {"bytes": b, "flops": 4 * pairs * c["nkh"] * group * c["hd"]}
    if c["op"] == "rope":
        t = c["tokens"]
        return {"bytes": t * (c["nqh"] * c["hd"] * 8 + c["nkh"] * c["hd"] * (8 + 4) + 4 * (c["axes"] + 2)),
                "flops": 6 * t * (c["nqh"] + c["nkh"]) * c["rot"] // 2}
    if c["op"] == "select":
        lists = c["layers"] * c["heads"]
        return {"bytes": 4 * lists * (sum(_counts(c)) + c["seqs"] * c["keep"]) + 8 * c["seqs"],
                "flops": 0}
    rows = c["layers"] * c["seqs"] * c["heads"] * c["n"]
    idx = c["seqs"] * c["n"] if c["accept"] else rows
    return {"bytes": 2 * rows * c["hd"] * 2 * 2 + 4 * idx + (0 if c["accept"] else 16 * rows), "flops": 0}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _cache(c, gen, layers, seqs, ctx, heads, hd, fill=True):
    """One half of a cache: [seq][layer][position][head][hd] or [seq][layer][head][position][hd]."""
    shape = (seqs, layers, heads, ctx, hd) if c["head_major"] else (seqs, layers, ctx, heads, hd)
    if not fill:
        return torch.zeros(shape, device=DEV, dtype=torch.float16)
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16)


def _tree(rng, tokens):
    """(who sees whom, depth) of a random tree of drafts, token 0 its root, parents before children."""
    sees = np.zeros((tokens, tokens), dtype=bool)
    depth = np.zeros(tokens, dtype=np.int64)
    for i in range(tokens):
        if i:
            p = int(rng.integers(max(0, i - 8), i))
            sees[i] = sees[p]
            depth[i] = depth[p] + 1
        sees[i, i] = True
    return sees, depth


def _words(sees):
    """Rows of truth values as rows of 32-bit words, bit j % 32 of word j / 32."""
    t = sees.shape[-1]
    pad = (-t) % 32
    bits = np.concatenate([sees, np.zeros(sees.shape[:-1] + (pad,), dtype=bool)], axis=-1)
    return np.packbits(bits, axis=-1, bitorder="little").view("<u4").astype(np.uint32)


def _dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=dtype))).to(DEV)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = {"case": c}
    if c["op"] == "attend":
        S, T, H, D = c["seqs"], c["tokens"], c["nkh"], c["hd"]
        nc, nt = _lengths(c)
        s["limit"] = max(n + t for n, t in zip(nc, nt))
        s["max_ctx"] = M = c["ctx"] + T + 13
        s["k"], s["v"] = (_cache(c, gen, 1, S, M, H, D) for _ in range(2))
        s["q"] = torch.randn((S, T, c["nqh"], D), generator=gen, device=DEV) * 1.5
        s["out"] = torch.zeros((S, T, c["nqh"], D), device=DEV)
        s["n_ctx"], s["n_tok"] = _dev(nc, np.int32), _dev(nt, np.int32)
        depth = np.tile(np.arange(T), (S, 1))
        s["mask"] = None
        if c["tree"]:
            trees = [_tree(rng, T) for _ in range(S)]
            depth = np.stack([d for _, d in trees])
            s["mask"] = _dev(_words(np.stack([m for m, _ in trees])).view(np.int32), np.int32)
        nc_ = np.asarray(nc)[:, None]
        s["k_pos"] = None
        if c["slots"] == "plain":
            q_pos = nc_ + depth
        elif c["slots"] == "padded":      # a left-padded prompt: the first slots hold nothing
            pad = rng.integers(0, max(1, c["ctx"] // 8) + 1, S)[:, None]
            k_pos = np.arange(M)[None] - pad
            q_pos = nc_ - pad + depth
            for i in range(S):
                k_pos[i, nc[i]:nc[i] + T] = q_pos[i, : T]
            s["k_pos"] = _dev(np.where(k_pos < 0, -1, k_pos), np.int32)
        else:                             # each head kept other positions of a longer context
            q_pos = 3 * nc_ + depth
            k_pos = np.cumsum(rng.integers(1, 4, (S, H, M)), axis=-1) - 1
            for i in range(S):
                k_pos[i, :, nc[i]:nc[i] + T] = q_pos[i, : T]
            s["k_pos"] = _dev(k_pos, np.int32)
        s["q_pos"] = _dev(q_pos, np.int32)
        s["slopes"] = None
        if c["slopes"]:                   # the usual geometric series over the heads, from 1/2 to 1/256
            s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, c["nqh"] + 1, device=DEV, dtype=torch.float32) / c["nqh"])
        if c["weights"]:
            s["weights_in"] = torch.rand((S, H, M), generator=gen, device=DEV) * 3
            s["weights_out"] = torch.zeros((S, H, M), device=DEV)
    elif c["op"] == "rope":
        n, S, A = c["tokens"], c["seqs"], c["axes"]
        s["max_ctx"] = c["ctx"] + 3
        s["q"] = torch.randn((n, c["nqh"], c["hd"]), generator=gen, device=DEV)
        s["k_new"], s["v_new"] = (torch.randn((n, c["nkh"], c["hd"]), generator=gen, device=DEV) for _ in range(2))
        s["q_out"] = torch.zeros_like(s["q"])
        s["k"], s["v"] = (_cache(c, gen, 1, S, s["max_ctx"], c["nkh"], c["hd"]) for _ in range(2))
        seq = np.arange(n) % S
        slot = np.empty(n, dtype=np.int64)
        for b in range(S):                # distinct slots, in no order
            slot[seq == b] = rng.permutation(s["max_ctx"])[: int((seq == b).sum())]
        text = np.arange(n) + int(rng.integers(0, c["far"] + 1))
        if A == 1:
            pos = text[:, None]
        else:                             # an image's grid: one time step, then rows and columns of patches
            side = max(1, int(math.sqrt(n)))
            pos = np.stack([text // side, text // side % side + int(text[0]), text % side, text % 7][:A], axis=1)
        s["pos"], s["seq"], s["slot"] = _dev(pos, np.int32), _dev(seq, np.int32), _dev(slot, np.int32)
        s["factors"] = [1.0 if i < c["rot"] // 4 else 1.0 + 7.0 * rng.random() for i in range(c["rot"] // 2)] if c["factors"] else None
    elif c["op"] == "select":
        L, S, H = c["layers"], c["seqs"], c["heads"]
        s["stride"] = c["n"] + 5
        w = torch.exp(2.5 * torch.randn((L, S, H, s["stride"]), generator=gen, device=DEV) - 6)
        # accumulated weights tie: what was never attended is 0, small sums meet on the same values
        w = torch.where(w < 2e-4, torch.zeros_like(w), w)
        s["scores"] = torch.where(w < 2e-2, torch.round(w * 4096) / 4096, w)
        s["n"] = _dev(_counts(c), np.int32)
        s["idx"] = torch.zeros((L, S, H, c["keep"]), device=DEV, dtype=torch.int32)
        s["count"] = torch.zeros((S,), device=DEV, dtype=torch.int32)
    else:
        L, S, H, n, D = c["layers"], c["seqs"], c["heads"], c["n"], c["hd"]
        if c["accept"]:                   # in place: the root stays, its descendants come from behind the accepted length
            T = 4 * n + 3
            s["max_ctx"] = s["dst_ctx"] = c["ctx"] + T + 1
            s["k"], s["v"] = (_cache(c, gen, L, S, s["max_ctx"], H, D) for _ in range(2))
            s["k_dst"], s["v_dst"] = s["k"], s["v"]
            path = np.stack([np.concatenate([[0], np.sort(rng.permutation(T - n)[: n - 1]) + n]) for _ in range(S)])
            s["idx"] = _dev(path, np.int32)
            s["count"] = _dev(rng.integers(1, n + 1, S) if S > 1 else [n], np.int32)
            s["base"] = _dev(rng.integers(c["ctx"] // 2, c["ctx"] + 1, S), np.int32)
        else:
            s["max_ctx"], s["dst_ctx"] = c["ctx"] + 1, n + 64
            s["k"], s["v"] = (_cache(c, gen, L, S, s["max_ctx"], H, D) for _ in range(2))
            s["k_dst"], s["v_dst"] = (_cache(c, gen, L, S, s["dst_ctx"], H, D, fill=False) for _ in range(2))
            keys = torch.rand((L, S, H, c["ctx"]), generator=gen, device=DEV)
            s["idx"] = keys.argsort(-1)[..., :n].sort(-1).values.to(torch.int32).contiguous()
            s["count"] = _dev([n] * S, np.int32)
            s["base"] = None
            s["w"] = torch.rand((L, S, H, s["max_ctx"]), generator=gen, device=DEV)
            s["p"] = torch.randint(0, 1 << 20, (L, S, H, s["max_ctx"]), generator=gen, device=DEV, dtype=torch.int32)
            s["w_dst"] = torch.zeros((L, S, H, s["dst_ctx"]), device=DEV)
            s["p_dst"] = torch.zeros((L, S, H, s["dst_ctx"]), device=DEV, dtype=torch.int32)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
_OWN = {}


def run(state):
    c = state["case"]
    if own:
        if "plan" not in state:           # the descriptors and the workspace that a program fills once and keeps
            state["plan"] = _PLAN[c["op"]](state)
        _CALL[c["op"]](state, state["plan"])
    else:
        _PLAIN[c["op"]](state)
    if c["op"] == "attend":
        return [state["out"], state["weights_out"]] if c["weights"] else [state["out"]]
    if c["op"] == "rope":
        return [state["q_out"], state["k"], state["v"]]
    if c["op"] == "select":
        return [state["idx"], state["count"]]
    if c["accept"]:
        return [state["k"], state["v"]]
    return [state["k_dst"], state["v_dst"], state["w_dst"], state["p_dst"]]


# ---- plain forms ----------------------------------------------------------
def _rows(cache, head_major):
    """A cache (without its layers) as [seq][head][position][hd]."""
    return cache if head_major else cache.transpose(1, 2)


def _plain_attend(s):
    c = s["case"]
    S, T, H, D, L = c["seqs"], c["tokens"], c["nkh"], c["hd"], s["limit"]
    G = c["nqh"] // H
    k, v = (_rows(s[x][:, 0], c["head_major"])[:, :, :L].float() for x in ("k", "v"))
    q = s["q"].view(S, T, H, G, D).permute(0, 2, 1, 3, 4).reshape(S, H, T * G, D)
    x = torch.matmul(q, k.transpose(-1, -2)).view(S, H, T, G, L) * (1.0 / math.sqrt(D))
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    slot = torch.arange(L, device=DEV)
    n_ctx, n_tok = s["n_ctx"].long().view(S, 1, 1), s["n_tok"].long().view(S, 1, 1)
    new = slot.view(1, 1, L) - n_ctx                                        # drafted token of each slot
    tok = torch.arange(T, device=DEV).view(1, T, 1)
    if s["mask"] is None:
        sees = new <= tok
    else:
        j = new.clamp(0, T - 1).expand(S, T, L)
        sees = ((torch.gather(s["mask"].long(), 2, j // 32) >> (j % 32)) & 1).bool()
    sees = torch.where(new < 0, torch.ones_like(sees), sees & (new < n_tok))   # [S][T][L]
    qp = s["q_pos"].long().view(S, 1, T, 1, 1)
    if s["k_pos"] is None:
        kp = torch.where(new[:, 0] < 0, slot.view(1, L), torch.gather(s["q_pos"].long(), 1, new[:, 0].clamp(0, T - 1)))
        kp = kp.view(S, 1, 1, 1, L)
    else:
        kp = s["k_pos"].long().view(S, -1, s["max_ctx"])[..., :L][:, :, None, None]
    ok = sees.view(S, 1, T, 1, L) & (kp >= 0)
    if c["window"]:
        ok = ok & (qp - kp < c["window"])
    if c["slopes"]:
        x = x + s["slopes"].view(1, H, 1, G, 1) * (kp - qp)
    x = torch.where(ok, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p.view(S, H, T * G, L), v).view(S, H, T, G, D).permute(0, 2, 1, 3, 4).reshape(S, T, c["nqh"], D)
    live = (tok < n_tok).view(S, T, 1, 1)
    s["out"].copy_(torch.where(live, o, s["out"]))
    if c["weights"]:
        w = (p * live.view(S, 1, T, 1, 1)).sum((2, 3))
        filled = (slot.view(1, 1, L) < n_ctx + n_tok)
        s["weights_out"][..., :L] = torch.where(filled, s["weights_in"][..., :L] + w, s["weights_out"][..., :L])


def _axis_of(c):
    """The position axis of each pair of dimensions: contiguous sections, or the axes in turn."""
    pairs, A = c["rot"] // 2, c["axes"]
    sec = _sections(c)
    if c["interleaved"]:
        return [i % A if i < A * sec[i % A] else 0 for i in range(pairs)]
    return [a for a in range(A) for _ in range(sec[a])]


def _sections(c):
    """Pairs of each axis: the later axes get an equal share, the first what is left."""
    pairs, A = c["rot"] // 2, c["axes"]
    rest = pairs * 5 // (16 * max(1, A - 2)) if A > 1 else 0
    return [pairs - (A - 1) * rest] + [rest] * (A - 1)


def _plain_rope(s):
    c = s["case"]
    R = c["rot"]
    pair = torch.arange(R // 2, device=DEV, dtype=torch.float64)
    freq = 10000.0 ** (-2.0 * pair / R)
    if s["factors"]:
        freq = freq / torch.tensor(s["factors"], device=DEV, dtype=torch.float32).double()
    pos = s["pos"].double()[:, torch.tensor(_axis_of(c), device=DEV)]
    ang = pos * freq                                                        # angles of far positions: 64 bits
    cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]

    def turn(x):
        y = x.clone()
        a, b = (x[..., : R // 2], x[..., R // 2: R]) if c["halves"] else (x[..., 0:R:2], x[..., 1:R:2])
        u, w = a * cos - b * sin, a * sin + b * cos
        if c["halves"]:
            y[..., : R // 2], y[..., R // 2: R] = u, w
        else:
            y[..., 0:R:2], y[..., 1:R:2] = u, w
        return y

    s["q_out"].copy_(turn(s["q"]))
    seq, slot = s["seq"].long(), s["slot"].long()
    k, v = (_rows(s[x][:, 0], c["head_major"]) for x in ("k", "v"))
    k[seq, :, slot] = turn(s["k_new"]).half()
    v[seq, :, slot] = s["v_new"].half()


def _plain_select(s):
    c = s["case"]
    keep, N = c["keep"], c["n"]
    n = s["n"].long().view(1, -1, 1, 1)
    at = torch.arange(N, device=DEV).view(1, 1, 1, N)
    x = s["scores"][..., :N]
    always = (at < c["first"]) | (at >= n - c["recent"])
    x = torch.where(always, torch.full_like(x, math.inf), x)
    x = torch.where(at < n, x, torch.full_like(x, -math.inf))
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices     # ties: the lower index first
    rank = torch.empty_like(order).scatter_(-1, order, at.expand_as(order))
    kept = (rank < keep) & (at < n)
    place = torch.where(kept, kept.long().cumsum(-1) - 1, torch.full_like(order, keep))
    idx = torch.full(x.shape[:-1] + (keep + 1,), -1, device=DEV, dtype=torch.int64)
    idx.scatter_(-1, place, at.expand_as(order))
    s["idx"].copy_(idx[..., :keep])
    s["count"].copy_(torch.minimum(s["n"], torch.full_like(s["n"], keep)))


def _plain_gather(s):
    c = s["case"]
    S, H, L, n, D = c["seqs"], c["heads"], c["layers"], c["n"], c["hd"]

    def view(x):                                                            # [seq][layer][head][position][hd]
        return x if c["head_major"] else x.transpose(2, 3)

    if c["accept"]:
        i = torch.arange(n, device=DEV).view(1, n)
        live = (i < s["count"].view(S, 1))
        src = (s["base"].view(S, 1) + s["idx"]).long().view(S, 1, 1, n, 1).expand(S, L, H, n, D)
        dst = (s["base"].view(S, 1) + i).long().view(S, 1, 1, n, 1).expand(S, L, H, n, D)
        for x in (view(s["k"]), view(s["v"])):
            rows = torch.where(live.view(S, 1, 1, n, 1), torch.gather(x, 3, src), torch.gather(x, 3, dst))
            x.scatter_(3, dst, rows)
        return
    at = s["idx"].long()                                                    # [layer][seq][head][n]: every list is full
    rows = at.permute(1, 0, 2, 3)[..., None].expand(S, L, H, n, D)
    view(s["k_dst"])[:, :, :, :n] = torch.gather(view(s["k"]), 3, rows)
    view(s["v_dst"])[:, :, :, :n] = torch.gather(view(s["v"]), 3, rows)
    s["w_dst"][..., :n] = torch.gather(s["w"], -1, at)
    s["p_dst"][..., :n] = torch.gather(s["p"], -1, at)


_PLAIN = {"attend": _plain_attend, "rope": _plain_rope, "select": _plain_select, "gather": _plain_gather}


# ---- this repository's calls ----------------------------------------------
def _vbs():
    if "vbs" not in _OWN:
        import vbs_b200
        _OWN["vbs"] = vbs_b200
    return _OWN["vbs"]


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _kv(s, k="k", v="v", ctx="max_ctx"):
    c = s["case"]
    heads, layers = c.get("nkh") or c["heads"], c.get("layers", 1)
    return _vbs().KvDesc(k=s[k].data_ptr(), v=s[v].data_ptr(), n_layers=layers, max_ctx=s[ctx], n_kv_heads=heads,
                         head_dim=c["hd"], n_seqs=c["seqs"], head_major=int(c["head_major"]),
                         seq_stride=layers * s[ctx] * heads * c["hd"])


def _plan_attend(s):
    c, vbs = s["case"], _vbs()
    kv = _kv(s)
    tree = vbs.TreeDesc(n_q_heads=c["nqh"], n_tokens=c["tokens"], scale=1.0 / math.sqrt(c["hd"]), softcap=c["cap"],
                        window=c["window"], ctx_limit=s["limit"], slopes=_ptr(s["slopes"]), n_ctx=_ptr(s["n_ctx"]),
                        n_tok=_ptr(s["n_tok"]), mask=_ptr(s["mask"]), q_pos=_ptr(s["q_pos"]), k_pos=_ptr(s["k_pos"]),
                        k_pos_per_head=int(c["slots"] == "evicted"), weights_in=_ptr(s.get("weights_in")),
                        weights_out=_ptr(s.get("weights_out")))
    work = torch.empty(max(1, vbs.tree_workspace(kv, tree)), dtype=torch.uint8, device=DEV)
    return kv, tree, work


def _call_attend(s, plan):
    kv, tree, work = plan
    _vbs().attention_tree(kv, 0, tree, s["q"].data_ptr(), s["out"].data_ptr(), work.data_ptr(), work.numel())


def _plan_rope(s):
    c, vbs = s["case"], _vbs()
    rope = vbs.rope_plan(c["hd"], rot_dim=c["rot"], theta=10000.0, halves=c["halves"], freq_factors=s["factors"],
                         sections=_sections(c) if c["axes"] > 1 else None, interleaved=c["interleaved"])
    return rope, _kv(s)


def _call_rope(s, plan):
    rope, kv = plan
    c = s["case"]
    _vbs().rope_store(rope, kv, 0, s["q"].data_ptr(), s["q_out"].data_ptr(), c["nqh"], s["k_new"].data_ptr(),
                      s["v_new"].data_ptr(), c["tokens"], s["pos"].data_ptr(), s["slot"].data_ptr(), seq=s["seq"].data_ptr())


def _call_select(s, plan):
    c = s["case"]
    _vbs().cache_select(s["scores"].data_ptr(), s["stride"], c["layers"], c["seqs"], c["heads"], s["n"].data_ptr(), c["n"],
                        c["keep"], c["first"], c["recent"], s["idx"].data_ptr(), s["count"].data_ptr())


def _plan_gather(s):
    c, vbs = s["case"], _vbs()
    n = c["n"]
    if c["accept"]:
        g = vbs.GatherDesc(n_max=n, idx=_ptr(s["idx"]), layer_stride=0, seq_stride=n, head_stride=0, count=_ptr(s["count"]),
                           src_base=_ptr(s["base"]), dst_base=_ptr(s["base"]))
    else:
        g = vbs.GatherDesc(n_max=n, idx=_ptr(s["idx"]), layer_stride=c["seqs"] * c["heads"] * n, seq_stride=c["heads"] * n,
                           head_stride=n, count=_ptr(s["count"]), weights_src=_ptr(s["w"]), weights_dst=_ptr(s["w_dst"]),
                           pos_src=_ptr(s["p"]), pos_dst=_ptr(s["p_dst"]))
    return _kv(s), _kv(s, "k_dst", "v_dst", "dst_ctx"), g


def _call_gather(s, plan):
    src, dst, g = plan
    _vbs().cache_gather(src, dst, g)


_PLAN = {"attend": _plan_attend, "rope": _plan_rope, "select": lambda s: None, "gather": _plan_gather}
_CALL = {"attend": _call_attend, "rope": _call_rope, "select": _call_select, "gather": _call_gather}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_attend(s):
    """Sequence by sequence and head by head, token by token where the mask differs."""
    c = s["case"]
    S, T, H, D = c["seqs"], c["tokens"], c["nkh"], c["hd"]
    G = c["nqh"] // H
    nc, nt = _lengths(c)
    out = s["out"].double()
    wout = s["weights_out"].double() if c["weights"] else None
    words = s["mask"].cpu().numpy().view(np.uint32) if s["mask"] is not None else None
    q_pos = s["q_pos"].cpu().numpy().astype(np.int64)
    k_pos = s["k_pos"].cpu().numpy().astype(np.int64) if s["k_pos"] is not None else None
    for b in range(S):
        n, t = nc[b], nt[b]
        end = n + t
        allowed = np.zeros((t, end), dtype=bool)
        allowed[:, :n] = True
        for i in range(t):
            for j in range(t):
                allowed[i, n + j] = (j <= i) if words is None else bool(int(words[b, i, j >> 5]) >> (j & 31) & 1)
        for h in range(H):
            if k_pos is None:
                where = np.concatenate([np.arange(n), q_pos[b, :t]])
            else:
                where = (k_pos[b, h] if k_pos.ndim == 3 else k_pos[b])[:end]
            far = q_pos[b, :t, None] - where[None]
            may = allowed & (where >= 0)[None]
            if c["window"]:
                may = may & (far < c["window"])
            kk = (s["k"][b, 0, h, :end] if c["head_major"] else s["k"][b, 0, :end, h]).double()
            vv = (s["v"][b, 0, h, :end] if c["head_major"] else s["v"][b, 0, :end, h]).double()
            may, far = torch.from_numpy(may).to(DEV), torch.from_numpy(far).to(DEV).double()
            for g in range(G):
                z = s["q"][b, :t, h * G + g].double() @ kk.T / math.sqrt(D)
                if c["cap"]:
                    z = c["cap"] * torch.tanh(z / c["cap"])
                if c["slopes"]:
                    z = z - float(s["slopes"][h * G + g]) * far
                z = z.masked_fill(~may, -math.inf)
                p = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)).masked_fill(~may, 0.0)
                out[b, :t, h * G + g] = p @ vv
                if wout is not None:
                    wout[b, h, :end] = (s["weights_in"][b, h, :end].double() if g == 0 else wout[b, h, :end]) + p.sum(0)
    return [out, wout] if c["weights"] else [out]


def _exact_rope(s):
    c = s["case"]
    R = c["rot"]
    axis = np.asarray(_axis_of(c))
    base = np.float64(10000.0) ** (-np.arange(0, R, 2) / np.float64(R))
    if s["factors"]:
        base = base / np.asarray(s["factors"], dtype=np.float32).astype(np.float64)
    ang = s["pos"].cpu().numpy().astype(np.float64)[:, axis] * base
    rot = torch.from_numpy(np.exp(1j * ang)).to(DEV)[:, None]

    def turned(x):
        y = x.double()
        first = slice(0, R // 2) if c["halves"] else slice(0, R, 2)
        second = slice(R // 2, R) if c["halves"] else slice(1, R, 2)
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * rot
        y[..., first], y[..., second] = z.real, z.imag
        return y

    k, v = s["k"].double(), s["v"].double()
    new_k, new_v = turned(s["k_new"]), s["v_new"].double()
    seq, slot = s["seq"].long(), s["slot"].long()
    if c["head_major"]:
        k[seq, 0, :, slot], v[seq, 0, :, slot] = new_k, new_v
    else:
        k[seq, 0, slot], v[seq, 0, slot] = new_k, new_v
    return [turned(s["q"]), k, v]


def _exact_gather(s):
    c = s["case"]
    L, S, H = c["layers"], c["seqs"], c["heads"]
    outs = [s[x].clone() for x in ("k_dst", "v_dst")]
    for src, dst in zip((s["k"], s["v"]), outs):
        for b in range(S):
            for l in range(L):
                for h in range(1 if c["accept"] else H):
                    n = int(s["count"][b])
                    base = int(s["base"][b]) if c["accept"] else 0
                    at = (s["idx"][b] if c["accept"] else s["idx"][l, b, h])[:n].long() + base
                    if c["accept"] and c["head_major"]:
                        dst[b, l, :, base:base + n] = src[b, l][:, at]
                    elif c["accept"]:
                        dst[b, l, base:base + n] = src[b, l][at]
                    elif c["head_major"]:
                        dst[b, l, h, :n] = src[b, l, h][at]
                    else:
                        dst[b, l, :n, h] = src[b, l, at, h]
    if c["accept"]:
        return outs
    w = torch.zeros_like(s["w_dst"])
    w[..., : c["n"]] = torch.take_along_dim(s["w"], s["idx"].long(), -1)
    return outs + [w, None]


def exact(case, seed):
    c = case
    if c["op"] == "select":               # whole numbers: equal or not
        return None
    if c["op"] == "attend" and c["seqs"] * c["nqh"] > 600:
        return None                       # too many heads one by one
    s = prepare(c, seed)
    return {"attend": _exact_attend, "rope": _exact_rope, "gather": _exact_gather}[c["op"]](s)
