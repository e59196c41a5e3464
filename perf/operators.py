"""The serving operators of a grouped-head text model (an 8-bit key/value cache: writing, attention, eviction; a linear
layer with 4-bit weights) as cases that can be timed and compared: the plain form of each in elementary torch
operations, and the call of sycl_minimax_h3_b200.ops that computes the same (``own``).

The cache: pages of 64 tokens, ``k``/``v`` int8 [pages, heads, 64, dim] with one float32 scale per page and head; the
tokens of a sequence that do not fill a page yet wait in its tail [sequences, heads, 64, dim] in the rows' own type.
``table`` int32 [sequences, width] names each sequence's pages, ``lens`` int32 [sequences] its tokens (those that a call
brings included), ``starts`` int32 [sequences + 1] its rows in the call's q, k, v.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ES = {"bf16": 2, "fp16": 2, "fp32": 4}
PAGE = 64
INF = float("inf")


# ---- the cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # writing to the cache: one step of a batch in the middle of its answers; prompts of unequal lengths
        {"name": "append_step", "op": "append", "dtype": "bf16", "B": 48, "new": 1, "lo": 1, "hi": 4096, "Hkv": 8, "D": 128},
        {"name": "append_prompt", "op": "append", "dtype": "fp16", "B": 3, "new": 4133, "lo": 700, "hi": 4133, "Hkv": 8, "D": 128},
        # attention over the cache: the first steps after a short prompt, one user
        {"name": "attend_one", "op": "attend", "dtype": "bf16", "B": 1, "new": 1, "lo": 77, "hi": 77, "Hq": 32, "Hkv": 8, "D": 128, "weights": False},
        # a step of a batch of unequal lengths
        {"name": "attend_batch", "op": "attend", "dtype": "bf16", "B": 48, "new": 1, "lo": 200, "hi": 8191, "Hq": 32, "Hkv": 8, "D": 128, "weights": False},
        # a step over one very long text
        {"name": "attend_long", "op": "attend", "dtype": "fp16", "B": 1, "new": 1, "lo": 131037, "hi": 131037, "Hq": 32, "Hkv": 8, "D": 128, "weights": False},
        # a part of a long prompt behind what is cached of it
        {"name": "attend_chunk", "op": "attend", "dtype": "fp16", "B": 1, "new": 1999, "lo": 17001, "hi": 17001, "Hq": 32, "Hkv": 8, "D": 128, "weights": False},
        # a step that also adds up the weight each token received, in float32 with 64-wide heads
        {"name": "attend_weights", "op": "attend", "dtype": "fp32", "B": 16, "new": 1, "lo": 100, "hi": 4500, "Hq": 16, "Hkv": 2, "D": 64, "weights": True},
        # eviction: one sequence that outgrew a small budget; a batch at a large one, some of it still within it
        {"name": "evict_one", "op": "evict", "dtype": "bf16", "B": 1, "lo": 1101, "hi": 1101, "budget": 512, "sinks": 4, "recent": 128, "Hkv": 8, "D": 128},
        {"name": "evict_batch", "op": "evict", "dtype": "bf16", "B": 12, "lo": 3500, "hi": 8111, "budget": 4096, "sinks": 4, "recent": 512, "Hkv": 8, "D": 128},
        # 4-bit linear layers: the qkv projection of a step; an odd layer with zero points; a batch's step through a wide layer
        {"name": "linear_one", "op": "linear", "dtype": "bf16", "M": 1, "N": 12288, "K": 4096, "group": 128, "sdtype": "bf16", "zero": False, "bias": False},
        {"name": "linear_odd", "op": "linear", "dtype": "fp32", "M": 3, "N": 1001, "K": 1368, "group": 32, "sdtype": "fp32", "zero": True, "bias": True},
        {"name": "linear_rows", "op": "linear", "dtype": "fp16", "M": 48, "N": 4096, "K": 14336, "group": 64, "sdtype": "fp16", "zero": False, "bias": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("append", "attend", "attend", "attend", "evict", "linear", "linear"))
    dtype = rng.choice(("bf16", "fp16", "fp32"))
    D = rng.choice((64, 128))
    Hkv = rng.choice((1, 2, 3, 4, 5, 8))
    if op == "append":
        B = _log(rng, 1, 48)
        if rng.random() < 0.5:
            return {"op": op, "dtype": dtype, "B": B, "new": 1, "lo": 1, "hi": _log(rng, 2, 4096), "Hkv": Hkv, "D": D}
        new = _log(rng, 2, max(3, 8000 // B))
        return {"op": op, "dtype": dtype, "B": B, "new": new, "lo": rng.randint(1, new), "hi": new, "Hkv": Hkv, "D": D}
    if op == "attend":
        per = rng.choice((1, 2, 3, 4, 7, 8, 16))
        if rng.random() < 0.7:
            B = _log(rng, 1, 48)
            hi = _log(rng, 1, 200000 // B)
            lo = rng.randint(max(1, hi // 8), hi)
            return {"op": op, "dtype": dtype, "B": B, "new": 1, "lo": lo, "hi": hi, "Hq": Hkv * per, "Hkv": Hkv, "D": D,
                    "weights": rng.random() < 0.4}
        B = _log(rng, 1, 4)
        new = _log(rng, 2, max(3, 1500 // B))
        hi = new + _log(rng, 1, max(2, 15000 // B))
        return {"op": op, "dtype": dtype, "B": B, "new": new, "lo": rng.randint(new, hi), "hi": hi, "Hq": Hkv * min(per, 4),
                "Hkv": Hkv, "D": D, "weights": rng.random() < 0.3}
    if op == "evict":
        B = _log(rng, 1, 12)
        hi = _log(rng, 130, 60000 // B)
        budget = PAGE * max(1, rng.randint(hi // 5, hi) // PAGE)
        recent = rng.randint(0, budget)
        return {"op": op, "dtype": dtype, "B": B, "lo": rng.randint(1, hi), "hi": hi, "budget": budget,
                "sinks": min(rng.choice((0, 1, 4)), budget - recent), "recent": recent, "Hkv": Hkv, "D": D}
    M = _log(rng, 1, 64)
    N = _log(rng, 16, 16000)
    K = 8 * _log(rng, 8, 1800)
    return {"op": op, "dtype": dtype, "M": M, "N": N, "K": K, "group": rng.choice((32, 64, 128, 0)),
            "sdtype": rng.choice(("bf16", "fp16", "fp32")), "zero": rng.random() < 0.4, "bias": rng.random() < 0.5}


def _spread(lo, hi, B):
    """B whole numbers over lo..hi, the same for every seed; the first is hi."""
    return [hi - int((hi - lo) * ((b * 0.6180339887) % 1.0)) for b in range(B)]


def _lens(case):
    return _spread(case["lo"], case["hi"], case["B"])


def _news(case):
    """New tokens of each sequence: one each, the whole prompt (append), or a part of at most ``new`` (attend)."""
    if case["new"] == 1:
        return [1] * case["B"]
    if case["op"] == "append":
        return _lens(case)
    return [min(n, l) for n, l in zip(_spread(max(1, case["new"] // 2), case["new"], case["B"]), _lens(case))]


def work(case):
    es = ES[case["dtype"]]
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        groups = -(-K // case["group"]) if case["group"] else 1
        b = N * K / 2 + groups * N * ES[case["sdtype"]] * (2 if case["zero"] else 1) + M * K * es + M * N * es + (4 * N if case["bias"] else 0)
        return {"bytes": b, "flops": 2.0 * M * N * K}
    L, h, D = _lens(case), case["Hkv"], case["D"]
    if case["op"] == "append":
        b = f = 0
        for n, l in zip(_news(case), L):
            full, part = l // PAGE - (l - n) // PAGE, l % PAGE
            old = (l - n) % PAGE if full else 0
            b += 2 * h * ((n + old) * D * es + full * (PAGE * D + 4) + min(part, n) * D * es)
            f += 2 * h * D * 3 * full * PAGE
        return {"bytes": float(b), "flops": float(max(f, 1))}
    if case["op"] == "evict":
        b = 0
        for l in L:
            if l > case["budget"]:
                b += h * (4 * l + case["budget"] * (2 * 2 * D + 4))
        return {"bytes": float(max(b, 8 * case["B"])), "flops": float(max(b, 1))}
    b = f = 0
    for n, l in zip(_news(case), L):
        full, part = l // PAGE, l % PAGE
        b += 2 * h * (full * (PAGE * D + 4) + part * D * es) + 2 * n * case["Hq"] * D * es + (8 * h * l if case["weights"] else 0)
        f += 4 * case["Hq"] * D * sum(range(l - n + 1, l + 1))
    return {"bytes": float(b), "flops": float(f)}


# ---- the inputs ------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        group = case["group"] or K
        groups = -(-K // group)
        codes = torch.randint(0, 16, (N, K), generator=g, device="cuda", dtype=torch.uint8)
        sd = DT[case["sdtype"]]
        scale = ((0.5 + torch.rand(groups, N, generator=g, device="cuda")) * (0.2 / math.sqrt(K))).to(sd)
        return {"case": case, "x": normal(M, K).to(dt), "codes": (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(),
                "scale": scale, "zero": (6 + 4 * torch.rand(groups, N, generator=g, device="cuda")).to(sd) if case["zero"] else None,
                "bias": normal(N) if case["bias"] else None, "out": torch.empty(M, N, dtype=dt, device="cuda"),
                "tiles": _tiles(codes)}
    B, h, D = case["B"], case["Hkv"], case["D"]
    L = _lens(case)
    W = max(l // PAGE for l in L) + 1
    st = {"case": case}
    spare = case["budget"] // PAGE if case["op"] == "evict" else 0
    P = B * spare + sum(l // PAGE for l in L) + 3
    # the pages of the sequences lie scattered; the ones that an eviction fills come first
    perm = (torch.randperm(P - B * spare, generator=g, device="cuda") + B * spare).to(torch.int32)
    meta = torch.full((B + B * W + B * spare,), -1, dtype=torch.int32, device="cuda")
    lens, table = meta[:B], meta[B:B + B * W].view(B, W)
    lens.copy_(torch.tensor(L, dtype=torch.int32))
    at = 0
    for b, l in enumerate(L):
        table[b, :l // PAGE] = perm[at:at + l // PAGE]
        at += l // PAGE
    if spare:
        meta[B + B * W:] = torch.arange(B * spare, dtype=torch.int32, device="cuda")
        st["spare"] = meta[B + B * W:].view(B, spare)
    st.update(meta=meta, meta0=meta.clone(), lens=lens, table=table, B=B, h=h, D=D, W=W, P=P)
    if case["op"] == "append":
        k = torch.zeros(P, h, PAGE, D, dtype=torch.int8, device="cuda")
        v, ks, vs = k.clone(), torch.zeros(P, h, device="cuda"), torch.zeros(P, h, device="cuda")
    else:
        k = (normal(P, h, PAGE, D) * 36).round().clamp(-127, 127).to(torch.int8)
        v = (normal(P, h, PAGE, D) * 36).round().clamp(-127, 127).to(torch.int8)
        ks = (0.6 + 0.8 * torch.rand(P, h, generator=g, device="cuda")) * (2.0 / 36)
        vs = (0.6 + 0.8 * torch.rand(P, h, generator=g, device="cuda")) / 36
    st.update(k=k, v=v, k_scale=ks, v_scale=vs, tail_k=(2 * normal(B, h, PAGE, D)).to(dt), tail_v=normal(B, h, PAGE, D).to(dt))
    if case["op"] == "evict" or case.get("weights"):
        wbuf = torch.zeros((P + B) * h * PAGE, device="cuda")
        # the weight that tokens gather is far from even: a few hold most of it, and many the same little
        wbuf.copy_((4 * normal(wbuf.numel()) - 4).exp2().clamp(max=64).mul(1024).floor().div(1024))
        st.update(wbuf=wbuf, wbuf0=wbuf.clone(), weight=wbuf[:P * h * PAGE].view(P, h, PAGE),
                  tail_weight=wbuf[P * h * PAGE:].view(B, h, PAGE))
    if case["op"] == "evict":
        n = B * spare
        st.update(k16=torch.empty(n, h, PAGE, D, dtype=torch.float16, device="cuda"),
                  v16=torch.empty(n, h, PAGE, D, dtype=torch.float16, device="cuda"), region=slice(0, n))
        return st
    news = _news(case)
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    T = starts[-1]
    st.update(starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), T=T, max_new=max(news), max_len=max(L))
    if case["op"] == "append":
        # k and v side by side, as a projection leaves them; k's channels have offsets of their own
        kv = normal(T, 2 * h * D)
        kv[:, :h * D] += 2 * normal(h * D)
        st["rows"] = kv.to(dt)
        done = [(b, j) for b, (n, l) in enumerate(zip(news, L)) for j in range((l - n) // PAGE, l // PAGE)]
        at = torch.tensor(done, dtype=torch.int64, device="cuda").view(-1, 2)
        st["done"] = table[at[:, 0], at[:, 1]].long()
        m = len(done)
        st.update(k16=torch.empty(m, h, PAGE, D, dtype=torch.float16, device="cuda"),
                  v16=torch.empty(m, h, PAGE, D, dtype=torch.float16, device="cuda"))
    else:
        st["Hq"] = case["Hq"]
        st["rows"] = normal(T, (case["Hq"] + 2 * h) * D).to(dt)
        st["out"] = torch.empty(T, case["Hq"] * D, dtype=dt, device="cuda")
    return st


def _tiles(codes):
    """The 4-bit weights as they are kept on the device: tiles of 16 outputs x 64 inputs, a lane (g, t) of 32 holding of
    outputs g and g + 8 the inputs 32 (w / 2) + 8 t + 4 (w % 2) + 0..3 in its word w; past the edges the code 8."""
    N, K = codes.shape
    c = torch.full((-(-N // 16) * 16, -(-K // 64) * 64), 8, dtype=torch.int64, device=codes.device)
    c[:N, :K] = codes
    c = c.view(c.shape[0] // 16, 2, 8, c.shape[1] // 64, 2, 4, 2, 2, 2)   # nt, row half, g, kt, w / 2, t, w % 2, pair, in pair
    half, pair, e = torch.meshgrid(*[torch.arange(2, device=codes.device)] * 3, indexing="ij")
    shift = 4 * (half + 2 * pair + 4 * e)
    word = (c.permute(0, 3, 2, 5, 4, 6, 1, 7, 8) << shift).sum((-1, -2, -3))                # nt, kt, g, t, w / 2, w % 2
    word = torch.where(word >= 1 << 31, word - (1 << 32), word)
    return word.to(torch.int32).reshape(c.shape[0], c.shape[3], 128)


# ---- one pass --------------------------------------------------------------------------------------------------------

def _cache(st):
    if "cache" not in st:
        from sycl_minimax_h3_b200 import ops

        st["cache"] = ops.KVCache(st["k"], st["v"], st["k_scale"], st["v_scale"], st["tail_k"], st["tail_v"], st["table"],
                                  st["lens"], st.get("weight"), st.get("tail_weight"))
    return st["cache"]


def run(state):
    return {"append": _append, "attend": _attend, "evict": _evict, "linear": _linear}[state["case"]["op"]](state)


def _append(st):
    h, D = st["h"], st["D"]
    if own:
        from sycl_minimax_h3_b200 import ops

        ops.kv_append(_cache(st), ops.Rows(st["rows"], 0, 2 * h * D, st["T"], h, D),
                      ops.Rows(st["rows"], h * D, 2 * h * D, st["T"], h, D), st["starts"], max_new=st["max_new"])
    else:
        _plain_append(st)
    out = {"tail_k": st["tail_k"], "tail_v": st["tail_v"]}
    if st["done"].numel():   # the pages that are full now, as the values that they stand for
        ks, vs = st["k_scale"][st["done"]], st["v_scale"][st["done"]]
        torch.mul(st["k"][st["done"]], ks[:, :, None, None], out=st["k16"])
        torch.mul(st["v"][st["done"]], vs[:, :, None, None], out=st["v16"])
        out.update(k=st["k16"], v=st["v16"], k_scale=ks, v_scale=vs)
    return out


def _quantise(x):
    """(codes, scales) of blocks x [..., 64, dim] in 64 bits: a value half way between two codes goes to the even one."""
    top = x.abs().amax((-1, -2))
    step = torch.where(top > 0, top, 1.0)[..., None, None]
    return (x * 127 / step).round().to(torch.int8), (top / 127).float()


def _plain_append(st):
    B, h, D = st["B"], st["h"], st["D"]
    n = (st["starts"][1:] - st["starts"][:-1]).long()
    new, old = st["lens"].long(), st["lens"].long() - n
    J = (st["max_new"] - 1) // PAGE + 2
    block = old[:, None] // PAGE + torch.arange(J, device="cuda")                      # [B, J]
    slot = block[..., None] * PAGE + torch.arange(PAGE, device="cuda")                 # [B, J, 64]
    row = (st["starts"][:-1].long()[:, None, None] + slot - old[:, None, None]).clamp(0, st["T"] - 1)
    fresh = (slot >= old[:, None, None]) & (slot < new[:, None, None])
    full = (block + 1) * PAGE <= new[:, None]
    page = st["table"].long().gather(1, block.clamp(max=st["W"] - 1))[full]
    rows = st["rows"].view(st["T"], 2, h, D)
    for_tail = fresh & ~full[..., None]
    b, j, i = for_tail.nonzero(as_tuple=True)

    def part(which, tail, codes, scales):
        x = rows[:, which][row].transpose(2, 3)                                        # [B, J, h, 64, D]
        x = torch.where(fresh[:, :, None, :, None], x, tail[:, None])
        codes[page], scales[page] = _quantise(x[full].double())
        tail[b, :, i] = x[b, j, :, i]

    part(0, st["tail_k"], st["k"], st["k_scale"])
    part(1, st["tail_v"], st["v"], st["v_scale"])


def _attend(st):
    case, h, D = st["case"], st["h"], st["D"]
    if case["weights"]:
        st["wbuf"].copy_(st["wbuf0"])
    if own:
        from sycl_minimax_h3_b200 import ops

        ops.attention_cached(ops.Rows(st["rows"], 0, (st["Hq"] + 2 * h) * D, st["T"], st["Hq"], D), _cache(st), st["starts"],
                             st["out"], max_new=st["max_new"], max_len=st["max_len"], accumulate=case["weights"])
    else:
        _plain_attend(st)
    return {"out": st["out"], "weight": st["wbuf"]} if case["weights"] else {"out": st["out"]}


def _plain_attend(st):
    B, h, D, W, Hq, T = st["B"], st["h"], st["D"], st["W"], st["Hq"], st["T"]
    page = st["table"].long().clamp(min=0)

    def values(codes, scales, tail):
        x = (codes[page] * scales[page][..., None, None]).transpose(1, 2).reshape(B, h, W * PAGE, D)
        return torch.cat((x, tail.float()), 2)

    k, v = values(st["k"], st["k_scale"], st["tail_k"]), values(st["v"], st["v_scale"], st["tail_v"])
    lens, starts = st["lens"].long(), st["starts"].long()
    whole = lens // PAGE * PAGE
    at = torch.arange(W * PAGE, device="cuda")
    slot = torch.cat((torch.where(at < whole[:, None], at, 1 << 40), whole[:, None] + torch.arange(PAGE, device="cuda")), 1)
    n = starts[1:] - starts[:-1]
    tok = torch.arange(T, device="cuda")
    seq = torch.searchsorted(starts, tok, right=True) - 1
    q = torch.zeros(B, st["max_new"], Hq, D, device="cuda")
    q[seq, tok - starts[seq]] = st["rows"][:, :Hq * D].reshape(T, Hq, D).float()
    q = q.view(B, st["max_new"], h, Hq // h, D).permute(0, 2, 3, 1, 4).reshape(B, h, -1, D)     # rows: head of the group, token
    i = torch.arange(st["max_new"], device="cuda")
    sees = slot[:, None] <= (lens - n)[:, None, None] + i[:, None]                               # [B, new, keys]
    sees = (sees & (i < n[:, None])[..., None])[:, None, None]
    s = (q @ k.transpose(2, 3)) / math.sqrt(D)
    s = s.view(B, h, Hq // h, st["max_new"], -1).masked_fill_(~sees, -INF)
    top = s.amax(-1, keepdim=True)
    p = (s - torch.where(top > -INF, top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    o = (p.view(B, h, -1, p.shape[-1]) @ v).view(B, h, Hq // h, st["max_new"], D).permute(0, 3, 1, 2, 4)
    st["out"].copy_(o[seq, tok - starts[seq]].reshape(T, Hq * D))
    if st["case"]["weights"]:
        w = p.sum((2, 3))                                                                        # [B, h, keys]
        used = (at[::PAGE] < whole[:, None])
        got = w[..., :W * PAGE].reshape(B, h, W, PAGE).transpose(1, 2)[used]
        st["weight"].index_put_((page[used],), got, accumulate=True)
        st["tail_weight"] += w[..., W * PAGE:]


def _evict(st):
    case = st["case"]
    st["meta"].copy_(st["meta0"])
    if own:
        from sycl_minimax_h3_b200 import ops

        ops.kv_evict(_cache(st), st["spare"], case["budget"], sinks=case["sinks"], recent=case["recent"])
    else:
        _plain_evict(st)
    r = st["region"]
    torch.mul(st["k"][r], st["k_scale"][r, :, None, None], out=st["k16"])
    torch.mul(st["v"][r], st["v_scale"][r, :, None, None], out=st["v16"])
    return {"k": st["k16"], "v": st["v16"], "k_scale": st["k_scale"][r], "v_scale": st["v_scale"][r],
            "weight": st["weight"][r], "meta": st["meta"]}


def _plain_evict(st):
    case, h, D, W = st["case"], st["h"], st["D"], st["W"]
    budget, keep = case["budget"], case["budget"] // PAGE
    over = st["lens"] > budget
    lens, page = st["lens"][over].long(), st["table"][over].long().clamp(min=0)
    B = lens.numel()
    whole = lens // PAGE * PAGE
    at = torch.arange(W * PAGE, device="cuda")
    slot = torch.cat((torch.where(at < whole[:, None], at, 1 << 40), whole[:, None] + torch.arange(PAGE, device="cuda")), 1)
    w = torch.cat((st["weight"][page].transpose(1, 2).reshape(B, h, W * PAGE), st["tail_weight"][over]), 2)
    kept = (slot < case["sinks"]) | (slot >= lens[:, None] - case["recent"])
    rank = torch.where(kept[:, None], INF, w).masked_fill((slot >= lens[:, None])[:, None], -INF)
    # the first of equals wins: a stable sort keeps their order
    idx = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget].sort(-1).values       # [B, h, budget]
    dst = st["spare"][over].long()

    def part(codes, scales, tail):
        x = torch.cat(((codes[page].double() * scales[page][..., None, None].double()).transpose(1, 2).reshape(B, h, W * PAGE, D),
                       tail[over].double()), 2)
        x = x.gather(2, idx[..., None].expand(-1, -1, -1, D)).view(B, h, keep, PAGE, D).transpose(1, 2)
        codes[dst], scales[dst] = _quantise(x)

    part(st["k"], st["k_scale"], st["tail_k"])
    part(st["v"], st["v_scale"], st["tail_v"])
    st["weight"][dst] = w.gather(2, idx).view(B, h, keep, PAGE).transpose(1, 2)
    old = st["table"][over, :keep]
    st["table"][over, :keep] = st["spare"][over]
    st["spare"][over] = old
    st["lens"].clamp_(max=budget)


def _linear(st):
    case = st["case"]
    if own:
        if "linear" not in st:
            from sycl_minimax_h3_b200 import ops

            st["linear"] = ops.Int4Linear(st["tiles"], st["scale"], case["N"], case["K"], case["group"], st["zero"], st["bias"])
        st["linear"].forward(st["x"], st["out"])
    else:
        N, K = case["N"], case["K"]
        codes = torch.stack((st["codes"] & 15, st["codes"] >> 4), 2).view(N, K).float()
        group = case["group"] or K
        at = torch.arange(K, device="cuda") // group
        zero = 8.0 if st["zero"] is None else st["zero"].float().t()[:, at]
        w = (codes - zero) * st["scale"].float().t()[:, at]
        y = st["x"].float() @ w.t()
        st["out"].copy_(y if st["bias"] is None else y + st["bias"])
    return st["out"]


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------

def _sequence(st, b, h0, codes, scales, tail, length):
    """Sequence b's cached rows of head h0 in 64 bits, [length, dim]."""
    full = length // PAGE
    pages = st["table"][b, :full].long()
    x = (codes[pages, h0].double() * scales[pages, h0].double()[:, None, None]).reshape(full * PAGE, st["D"])
    return torch.cat((x, tail[b, h0, :length - full * PAGE].double()))


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear":
        w = torch.empty(case["N"], case["K"], dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (st["codes"] % 16).double(), (st["codes"] // 16).double()
        group = case["group"] or case["K"]
        for i in range(st["scale"].shape[0]):
            cols = slice(i * group, (i + 1) * group)
            w[:, cols] -= 8 if st["zero"] is None else st["zero"][i].double()[:, None]
            w[:, cols] *= st["scale"][i].double()[:, None]
        y = torch.einsum("mk,nk->mn", st["x"].double(), w)
        return y + st["bias"].double() if case["bias"] else y
    B, h, D, L = st["B"], st["h"], st["D"], _lens(case)
    if case["op"] == "append":
        tails = {"tail_k": st["tail_k"].double(), "tail_v": st["tail_v"].double()}
        vals, steps = {"k": [], "v": []}, {"k_scale": [], "v_scale": []}
        first = st["starts"].tolist()
        for b, (n, l) in enumerate(zip(_news(case), L)):
            for name, off in (("k", 0), ("v", h * D)):
                new = st["rows"][first[b]:first[b] + n, off:off + h * D].double().view(n, h, D).transpose(0, 1)
                tail = tails["tail_" + name]
                open_ = (l - n) % PAGE
                all_ = torch.cat((tail[b, :, :open_], new), 1)
                full = all_.shape[1] // PAGE
                for j in range(full):
                    blk = all_[:, j * PAGE:(j + 1) * PAGE]
                    top = blk.abs().flatten(1).max(1).values
                    vals[name].append(torch.round(blk * 127 / top[:, None, None]) * (top / 127)[:, None, None])
                    steps[name + "_scale"].append(top / 127)
                rest = all_[:, full * PAGE:]
                tail[b, :, :rest.shape[1]] = rest
        out = dict(tails)
        if vals["k"]:
            out.update({m: torch.stack(x) for m, x in {**vals, **steps}.items()})
        return out
    if case["op"] == "attend":
        out = torch.zeros(st["T"], case["Hq"], D, dtype=torch.float64, device="cuda")
        weight = st["wbuf0"].double() if case["weights"] else None
        first = st["starts"].tolist()
        per = case["Hq"] // h
        for b, (n, l) in enumerate(zip(_news(case), L)):
            mask = torch.arange(l, device="cuda")[None] > torch.arange(l - n, l, device="cuda")[:, None]
            for kv in range(h):
                k = _sequence(st, b, kv, st["k"], st["k_scale"], st["tail_k"], l)
                v = _sequence(st, b, kv, st["v"], st["v_scale"], st["tail_v"], l)
                total = torch.zeros(l, dtype=torch.float64, device="cuda")
                for hq in range(kv * per, kv * per + per):
                    q = st["rows"][first[b]:first[b] + n, hq * D:(hq + 1) * D].double()
                    p = torch.softmax((q @ k.t() / D ** 0.5).masked_fill(mask, -INF), 1)
                    out[first[b]:first[b] + n, hq] = p @ v
                    total += p.sum(0)
                if weight is not None:
                    full = l // PAGE
                    pages = st["table"][b, :full].long()
                    weight[:st["P"] * h * PAGE].view(-1, h, PAGE)[pages, kv] += total[:full * PAGE].view(full, PAGE)
                    weight[st["P"] * h * PAGE:].view(B, h, PAGE)[b, kv, :l - full * PAGE] += total[full * PAGE:]
        out = out.view(st["T"], -1)
        return {"out": out, "weight": weight} if case["weights"] else {"out": out}
    # evict
    keep = case["budget"] // PAGE
    r = st["region"]
    res = {"k": st["k"][r].double() * st["k_scale"][r, :, None, None].double(),
           "v": st["v"][r].double() * st["v_scale"][r, :, None, None].double(), "k_scale": st["k_scale"][r].double(),
           "v_scale": st["v_scale"][r].double(), "weight": st["weight"][r].double(), "meta": None}
    for b, l in enumerate(L):
        if l <= case["budget"]:
            continue
        full = l // PAGE
        pages, to = st["table"][b, :full].long(), st["spare"][b].long()
        for kv in range(h):
            w = torch.cat((st["weight"][pages, kv].reshape(-1), st["tail_weight"][b, kv, :l - full * PAGE])).double()
            order = w.clone()
            order[:case["sinks"]] = INF
            order[l - case["recent"]:] = INF
            idx = torch.argsort(-order, stable=True)[:case["budget"]].sort().values
            res["weight"][to, kv] = w[idx].view(keep, PAGE)
            for name in ("k", "v"):
                x = _sequence(st, b, kv, st[name], st[name + "_scale"], st["tail_" + name], l)[idx].view(keep, PAGE, D)
                top = x.abs().flatten(1).max(1).values
                res[name + "_scale"][to, kv] = top / 127
                res[name][to, kv] = torch.round(x * 127 / top[:, None, None]) * (top / 127)[:, None, None]
    return res
