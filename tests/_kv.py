"""The 8-bit key/value cache for the tests: caches with given contents, and the definitions in 64 bits."""
from __future__ import annotations

import torch

from sycl_minimax_h3_b200 import ops

PAGE = ops.PAGE


def rows(t: torch.Tensor, heads: int, dim: int, offset: int = 0) -> ops.Rows:
    """Rows at element ``offset`` of every row of a [tokens, width] tensor."""
    return ops.Rows(t, offset, t.shape[1], t.shape[0], heads, dim)


def starts_of(news, device) -> torch.Tensor:
    s = [0]
    for n in news:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device=device)


def random_cache(lens, heads, dim, dtype, device, seed=0, weights=False, extra=3, width=None) -> ops.KVCache:
    """A cache whose sequences have these lengths, with random codes, scales and tails, its pages in random order."""
    g = torch.Generator().manual_seed(seed)
    full = [l // PAGE for l in lens]
    pages = sum(full) + extra
    c = ops.KVCache.empty(pages, len(lens), width or max(full) + 1, heads, dim, dtype, device, weights)
    c.k.copy_(torch.randn(c.k.shape, generator=g).mul(36).round().clamp(-127, 127))
    c.v.copy_(torch.randn(c.k.shape, generator=g).mul(36).round().clamp(-127, 127))
    c.k_scale.copy_(0.03 + 0.06 * torch.rand(c.k_scale.shape, generator=g))
    c.v_scale.copy_(0.01 + 0.04 * torch.rand(c.v_scale.shape, generator=g))
    c.tail_k.copy_(torch.randn(c.tail_k.shape, generator=g) * 2)
    c.tail_v.copy_(torch.randn(c.tail_v.shape, generator=g))
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    at = 0
    for b, n in enumerate(full):
        c.table[b, :n] = perm[at:at + n]
        at += n
    c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    if weights:
        c.weight.copy_(torch.rand(c.weight.shape, generator=g))
        c.tail_weight.copy_(torch.rand(c.tail_weight.shape, generator=g))
    return c


def sequence(c: ops.KVCache, b: int, which: str) -> torch.Tensor:
    """The keys or values of sequence b in 64 bits on the CPU, [lens[b], heads, dim]."""
    n = int(c.lens[b])
    full = n // PAGE
    pages = c.table[b, :full].long()
    codes, scale, tail = getattr(c, which), getattr(c, which + "_scale"), getattr(c, "tail_" + which)
    x = codes[pages].double() * scale[pages].double()[..., None, None]          # [full, heads, 64, dim]
    x = x.transpose(1, 2).reshape(full * PAGE, codes.shape[1], codes.shape[3])
    return torch.cat((x, tail[b, :, :n - full * PAGE].double().transpose(0, 1))).cpu()


def seq_weights(c: ops.KVCache, b: int) -> torch.Tensor:
    """[heads, lens[b]] weights of sequence b on the CPU."""
    n = int(c.lens[b])
    full = n // PAGE
    w = c.weight[c.table[b, :full].long()].transpose(0, 1).reshape(c.k.shape[1], full * PAGE)
    return torch.cat((w, c.tail_weight[b, :, :n - full * PAGE]), 1).cpu()


def quantised(x: torch.Tensor):
    """(codes, scale) of a block x [64, dim] (any shape) in 64 bits: the largest finite magnitude takes 127, a value half way
    between two codes the even one, an infinity +-127, a NaN 0."""
    x = x.double()
    fin = torch.where(x.isfinite(), x, 0.0)
    top = fin.abs().max()
    scale = (top / 127).float()
    if top == 0:
        return torch.zeros_like(x, dtype=torch.int8), scale
    q = (fin * 127 / top).round()
    q = torch.where(x == float("inf"), 127.0, torch.where(x == -float("inf"), -127.0, q))
    return q.to(torch.int8), scale


def attention(c: ops.KVCache, q: torch.Tensor, heads_q: int, starts):
    """(out, weights, bound): softmax(q k^T / sqrt(dim)) v of every sequence in 64 bits; the weights that each sequence's
    slots received, [heads, lens[b]] each; and for every output the most that arithmetic in 32 bits may be off:

    sum_j p_j |v_j| times
      2 ds     the relative error of p by an error ds of its score (once in p, once in the sum of all p), with
               ds <= (dim + 8) 2^-23 max_j sum_d |q_d k_jd| / sqrt(dim): a 32-bit sum of dim products that may cut off
               instead of rounding, and the factors' roundings
      pr       the rounding of p itself: half a step of fp16, 2^-11, where the rows are 16-bit; 2^-21 where two terms of
               fp16 stand for p (float32); 2^-22 of the exponential
      (L / 16 + 64) 2^-23   the sums over L keys, of which a lane adds every sixteenth one after the other
    (in float32 also 2^-21 of |q k| for the scores: q enters as two terms). And sum_j |v_j| times 2^-38: p is held as fp16
    between 2^-24 and 2^14, the row's largest, so one of its smallest numbers is off by half of 2^-24, which is 2^-39 of the
    largest p and of the sum of all p at most; twice that for the two terms. Where many rows come in a call, p times its
    page's scale is what is rounded, its largest at least 2^6: 2^-31 of the row's largest p scale for every code |v| / scale,
    twice that for the reference's own move (the tail's scale is the power of two that brings its largest into [2^13,
    2^14)). Then half a step of the output's type, of
    what is rounded: the value and the errors before it."""
    heads, dim = c.k.shape[1], c.k.shape[3]
    starts = starts.tolist()
    T = q.shape[0]
    qd = q.double().cpu().view(T, heads_q, dim)
    out = torch.zeros(T, heads_q, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    weights = []
    wide = c.tail_k.dtype == torch.float32
    for b in range(len(starts) - 1):
        n, L = starts[b + 1] - starts[b], int(c.lens[b])
        k, v = sequence(c, b, "k"), sequence(c, b, "v")
        w = torch.zeros(heads, L, dtype=torch.float64)
        full = L // PAGE
        page = c.v_scale[c.table[b, :full].long()].double().cpu()
        top = torch.where(c.tail_v[b].isfinite(), c.tail_v[b], 0).double().abs().amax((1, 2)).cpu() if L % PAGE else torch.ones(heads)
        vscale = torch.cat((page.repeat_interleave(PAGE, 0), (2.0 ** (torch.floor(torch.log2(top)) - 13)).expand(L % PAGE, heads)))
        pos = torch.arange(L - n, L)
        hidden = torch.arange(L)[None] > pos[:, None]
        for h in range(heads_q):
            kh, vh = k[:, h // (heads_q // heads)], v[:, h // (heads_q // heads)]
            x = qd[starts[b]:starts[b + 1], h]
            s = (x @ kh.T / dim ** 0.5).masked_fill(hidden, -float("inf"))
            p = torch.nan_to_num(torch.softmax(s, 1)) if L else torch.zeros(n, 0, dtype=torch.float64)
            out[starts[b]:starts[b + 1], h] = p @ vh
            w[h // (heads_q // heads)] += p.sum(0)
            mag = (x.abs() @ kh.abs().T / dim ** 0.5).masked_fill(hidden, 0.0)
            ds = (mag.max(1).values if L else torch.zeros(n)) * ((dim + 8) * 2.0 ** -23 + (2.0 ** -21 if wide else 0.0))
            rel = 2 * ds + (2.0 ** -21 if wide else 2.0 ** -11) + 2.0 ** -22 + (L / 16 + 64) * 2.0 ** -23
            bound[starts[b]:starts[b + 1], h] = rel[:, None] * (p @ vh.abs()) + 2.0 ** -38 * ((~hidden).double() @ vh.abs())
            if not wide and L:
                vs = vscale[:, h // (heads_q // heads)]
                code = torch.where(vs[:, None] > 0, vh.abs() / torch.where(vs > 0, vs, 1)[:, None], 0)
                bound[starts[b]:starts[b + 1], h] += 2.0 ** -30 * (p * vs).max(1, keepdim=True).values * ((~hidden).double() @ code)
        weights.append(w)
    half = torch.finfo(c.tail_k.dtype).eps / 2
    bound = bound + half * (out.abs() + bound) + torch.finfo(c.tail_k.dtype).tiny
    return out.reshape(T, -1), weights, bound.reshape(T, -1)
