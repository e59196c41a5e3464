"""The 8-bit key/value cache on the GPU: h3s_kv_append, h3s_attention_cached and h3s_kv_evict against their definitions in
64 bits (tests/_kv.py). Codes, scales, kept tokens, tables and lengths have to be equal; outputs may be off by what the
arithmetic's roundings add up to (``_kv.attention``) and half a step of their own type."""
import pytest
import torch

import _kv
from _kv import PAGE
from sycl_minimax_h3_b200 import native, ops

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def wait(device):
    ops.context(device).wait()


def make_rows(T, width, dtype, device, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, width, generator=g) * 1.5 + torch.randn(width, generator=g)
    return x.to(dtype).to(device)


# ---- writing ----

def fill(cache, news, k, v, dim, device, table=True):
    """Appends news[b] rows to every sequence of a cache whose table gives out pages in a scattered order."""
    cache.lens.add_(torch.tensor(news, dtype=torch.int32, device=device))
    heads = cache.k.shape[1]
    ops.kv_append(cache, _kv.rows(k, heads, dim), _kv.rows(v, heads, dim), _kv.starts_of(news, device))


def scatter_table(cache, device, seed=0):
    seqs, width = cache.table.shape
    g = torch.Generator().manual_seed(seed)
    cache.table.copy_(torch.randperm(cache.k.shape[0], generator=g)[:seqs * width].view(seqs, width))


def check_written(cache, b, heads, want_k, want_v):
    """Sequence b holds exactly the rows want_* [tokens, heads, dim]: full blocks quantised, the rest as it is."""
    n = want_k.shape[0]
    assert int(cache.lens[b]) == n
    for name, want in (("k", want_k.cpu()), ("v", want_v.cpu())):
        for j in range(n // PAGE):
            page = int(cache.table[b, j])
            for h in range(heads):
                codes, scale = _kv.quantised(want[j * PAGE:(j + 1) * PAGE, h])
                assert torch.equal(getattr(cache, name + "_scale")[page, h].cpu(), scale), (name, b, j, h)
                assert torch.equal(getattr(cache, name)[page, h].cpu(), codes), (name, b, j, h)
        tail = getattr(cache, "tail_" + name)[b, :, :n % PAGE].cpu().transpose(0, 1)
        assert torch.equal(tail.view(torch.uint8), want[n // PAGE * PAGE:].contiguous().view(torch.uint8)), (name, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dim,news", [(1, 64, [1]), (2, 128, [64]), (3, 64, [63, 0, 65, 200]), (2, 128, [130, 1, 64, 0])])
def test_append_from_empty(dtype, heads, dim, news, cuda):
    k, v = make_rows(sum(news), heads * dim, dtype, cuda, 1), make_rows(sum(news), heads * dim, dtype, cuda, 2)
    cache = ops.KVCache.empty(4 * len(news) + 2, len(news), 4, heads, dim, dtype, cuda)
    scatter_table(cache, cuda)
    fill(cache, news, k, v, dim, cuda)
    wait(cuda)
    at = 0
    for b, n in enumerate(news):
        check_written(cache, b, heads, k[at:at + n].view(n, heads, dim), v[at:at + n].view(n, heads, dim))
        at += n


@pytest.mark.parametrize("dtype", TYPES)
def test_append_does_not_depend_on_the_pieces(dtype, cuda):
    """150 tokens of two sequences in pieces of many sizes (also one at a time over a page's end) leave the same bits."""
    heads, dim, n = 2, 64, 150
    k, v = make_rows(n, heads * dim, dtype, cuda, 3), make_rows(n, heads * dim, dtype, cuda, 4)
    caches = []
    for pieces in ([150], [1] * 150, [63, 1, 1, 85], [64, 64, 22], [60, 70, 20], [10, 120, 20]):
        cache = ops.KVCache.empty(8, 2, 3, heads, dim, dtype, cuda, weights=True)
        scatter_table(cache, cuda)
        at = 0
        for p in pieces:
            both = torch.cat((k[at:at + p], v[at:at + p]))     # sequence 0 gets the k rows as k, sequence 1 the v rows
            fill(cache, [p, p], both, both, dim, cuda)
            at += p
        wait(cuda)
        check_written(cache, 0, heads, k.view(n, heads, dim), k.view(n, heads, dim))
        caches.append(cache)
    for c in caches[1:]:
        for name in ("k", "v", "k_scale", "v_scale", "tail_k", "tail_v"):
            a, b = getattr(caches[0], name), getattr(c, name)
            if name.startswith("tail"):
                a, b = a[:, :, :n % PAGE], b[:, :, :n % PAGE]
            else:
                used = caches[0].table[:, :n // PAGE].reshape(-1).long()
                a, b = a[used], b[used]
            assert torch.equal(a, b), name


@pytest.mark.parametrize("dtype", TYPES)
def test_append_reads_strided_and_unaligned_rows(dtype, cuda):
    """k and v inside a wider buffer, at an odd element offset, and more rows in it than the sequences have."""
    heads, dim, n = 2, 64, 70
    buf = make_rows(n + 3, 2 * heads * dim + 7, dtype, cuda, 5)
    cache = ops.KVCache.empty(3, 1, 2, heads, dim, dtype, cuda)
    scatter_table(cache, cuda)
    cache.lens.fill_(n)
    for off in (0, 3):
        kr = ops.Rows(buf, off, buf.shape[1], n + 3 - (off > 0), heads, dim)
        vr = ops.Rows(buf, off + heads * dim, buf.shape[1], n + 3 - (off > 0), heads, dim)
        ops.kv_append(cache, kr, vr, _kv.starts_of([n], cuda))
        wait(cuda)
        at = lambda o: buf[:n, o:o + heads * dim].reshape(n, heads, dim)  # noqa: E731
        check_written(cache, 0, heads, at(off), at(off + heads * dim))


@pytest.mark.parametrize("dtype", TYPES)
def test_append_edge_values(dtype, cuda):
    """Zeros, infinities, NaN, the type's largest and smallest values, and values half way between two codes."""
    heads, dim = 5, 64
    x = torch.randn(PAGE, heads, dim, generator=torch.Generator().manual_seed(6)).to(dtype)
    info = torch.finfo(dtype)
    x[:, 0] = 0
    x[3, 1, 5], x[4, 1, 6], x[5, 1, 7] = float("inf"), -float("inf"), float("nan")
    x[:, 2] *= info.tiny
    x[0, 3] = info.max
    x[1, 3] = -info.max / 2
    # the largest 127: the halves lie half way between two codes
    x[:, 4] = (torch.arange(PAGE * dim).view(PAGE, dim) % 253 - 126).to(dtype) / 2
    x[0, 4, 0] = 127
    x = x.reshape(PAGE, heads * dim).to(cuda)
    cache = ops.KVCache.empty(1, 1, 1, heads, dim, dtype, cuda)
    cache.table.zero_()
    fill(cache, [PAGE], x, x, dim, cuda)
    wait(cuda)
    check_written(cache, 0, heads, x.view(PAGE, heads, dim), x.view(PAGE, heads, dim))
    nothing = torch.full_like(x, float("nan"))
    cache.lens.zero_()
    fill(cache, [PAGE], nothing, nothing, dim, cuda)
    wait(cuda)
    assert not cache.k.any() and not cache.k_scale.any()


def test_append_weights_move_with_their_tokens(cuda):
    heads, dim = 2, 64
    x = make_rows(70, heads * dim, torch.float16, cuda, 7)
    cache = ops.KVCache.empty(2, 1, 2, heads, dim, torch.float16, cuda, weights=True)
    cache.table.copy_(torch.tensor([[1, 0]]))
    cache.weight.fill_(9)
    cache.tail_weight.fill_(9)
    fill(cache, [30], x[:30], x[:30], dim, cuda)
    wait(cuda)
    assert not cache.tail_weight[0, :, :30].any()
    cache.tail_weight[0, :, :30] = torch.arange(60, device=cuda).view(2, 30).float()
    fill(cache, [40], x[30:].contiguous(), x[30:].contiguous(), dim, cuda)
    wait(cuda)
    assert torch.equal(cache.weight[1, :, :30], torch.arange(60, device=cuda).view(2, 30).float())
    assert not cache.weight[1, :, 30:].any() and not cache.tail_weight[0, :, :6].any()
    assert bool((cache.weight[0] == 9).all())


# ---- attention ----

def check_attention(cache, q, starts, out, Hq):
    want, weights, bound = _kv.attention(cache, q, Hq, starts)
    got = out.double().cpu()
    off = (got - want).abs() - bound
    assert not got.isnan().any()
    assert float(off.max()) <= 0, f"off by {float(off.max()):.3g} more than the roundings"
    return weights


def run_attention(cache, q, Hq, starts, device, **kw):
    dim = cache.k.shape[3]
    out = torch.full((q.shape[0], Hq * dim), 7.0, dtype=q.dtype, device=device)
    ops.attention_cached(_kv.rows(q, Hq, dim), cache, starts, out, **kw)
    wait(device)
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,per,lens,news", [
    (1, 1, [1], [1]),
    (2, 4, [63, 64, 65, 1], [1, 1, 1, 1]),
    (2, 16, [700], [1]),
    (1, 3, [5, 0, 200, 64], [5, 0, 7, 64]),
    (2, 5, [130, 3], [130, 0]),
    (1, 8, [3000, 40], [1, 1]),
    (3, 2, [257, 300, 128], [33, 1, 100]),
])
def test_attention(dtype, dim, heads, per, lens, news, cuda):
    cache = _kv.random_cache(lens, heads, dim, dtype, cuda, seed=len(lens) + dim)
    q = make_rows(sum(news), heads * per * dim, dtype, cuda, 8)
    starts = _kv.starts_of(news, cuda)
    out = run_attention(cache, q, heads * per, starts, cuda)
    check_attention(cache, q, starts, out, heads * per)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seqs", [1, 5, 40, 300])
@pytest.mark.parametrize("heads,per", [(1, 4), (5, 2), (1, 9)])
def test_attention_shares_of_many_sequences(dtype, seqs, heads, per, cuda):
    """Sequences of all lengths in one call, several to a lane and to a CTA's share, some with nothing new, and one that is
    much longer than the others."""
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, 400, (seqs,), generator=g).tolist()
    lens[seqs // 2] = 6000 if seqs <= 40 else 20000
    news = [1 if b % 7 != 3 else 0 for b in range(seqs)]
    news[seqs // 2] = 1
    cache = _kv.random_cache(lens, heads, 64, dtype, cuda, seed=seqs + heads)
    q = make_rows(sum(news), heads * per * 64, dtype, cuda, 48)
    starts = _kv.starts_of(news, cuda)
    out = run_attention(cache, q, heads * per, starts, cuda, max_new=1)
    check_attention(cache, q, starts, out, heads * per)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("max_new,max_len", [(1, 1), (1, 100000), (40, 64), (1000, 1 << 40)])
def test_attention_hints_only_divide_the_work(dtype, max_new, max_len, cuda):
    lens, news, heads, per, dim = [900, 333, 70], [40, 1, 70], 2, 3, 128
    cache = _kv.random_cache(lens, heads, dim, dtype, cuda, seed=9)
    q = make_rows(sum(news), heads * per * dim, dtype, cuda, 10)
    starts = _kv.starts_of(news, cuda)
    out = run_attention(cache, q, heads * per, starts, cuda, max_new=max_new, max_len=max_len)
    check_attention(cache, q, starts, out, heads * per)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_rows_that_see_nothing_and_rows_behind_the_last(dtype, cuda):
    """More new rows than tokens: the first rows see nothing and come out 0. Rows behind starts[seqs] stay as they were."""
    lens, news, heads, per, dim = [2, 0, 70], [6, 3, 1], 2, 2, 64
    cache = _kv.random_cache(lens, heads, dim, dtype, cuda, seed=11)
    q = make_rows(sum(news) + 4, heads * per * dim, dtype, cuda, 12)
    starts = _kv.starts_of(news, cuda)
    out = run_attention(cache, q, heads * per, starts, cuda)
    n = sum(news)
    check_attention(cache, q[:n], starts, out[:n], heads * per)
    assert not out[:4].any() and not out[6:9].any()
    assert bool((out[n:] == 7).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_reads_strided_and_unaligned_queries(dtype, cuda):
    heads, per, dim, n = 2, 2, 64, 3
    cache = _kv.random_cache([150], heads, dim, dtype, cuda, seed=13)
    buf = make_rows(n, heads * per * dim + 5, dtype, cuda, 14)
    starts = _kv.starts_of([n], cuda)
    for off in (0, 5):
        out = torch.empty(n, heads * per * dim, dtype=dtype, device=cuda)
        ops.attention_cached(ops.Rows(buf, off, buf.shape[1], n, heads * per, dim), cache, starts, out)
        wait(cuda)
        check_attention(cache, buf[:, off:off + heads * per * dim], starts, out, heads * per)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1e-30, 1e-5, 1.0, 3e4, 1e30])
def test_attention_query_sizes(dtype, size, cuda):
    """Queries of any size the type has, against keys whose scores stay moderate: q is brought to fp16 by a power of two."""
    if dtype == torch.float16 and not 1e-6 < size < 6e4:
        pytest.skip("outside fp16")
    heads, per, dim = 1, 2, 64
    cache = _kv.random_cache([200], heads, dim, dtype, cuda, seed=15)
    q = torch.randn(1, heads * per * dim, generator=torch.Generator().manual_seed(16)).clamp(-1.5, 1.5).mul(size).to(dtype).to(cuda)
    cache.k_scale.div_(size)
    cache.tail_k.zero_()
    starts = _kv.starts_of([1], cuda)
    out = run_attention(cache, q, heads * per, starts, cuda)
    check_attention(cache, q, starts, out, heads * per)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_hidden_slots_may_hold_anything(dtype, cuda):
    """What lies behind a sequence's end, or behind a query's own slot, does not reach the output: NaN and infinities in
    the tail's unused rows and in later tokens, and infinite scales of pages that are not the sequence's."""
    heads, per, dim = 2, 2, 64
    cache = _kv.random_cache([100], heads, dim, dtype, cuda, seed=17)
    cache.tail_k[0, :, 36:] = float("nan")
    cache.tail_v[0, :, 36:] = float("inf")
    others = [p for p in range(cache.k.shape[0]) if p != int(cache.table[0, 0])]
    cache.k_scale[others] = float("nan")
    cache.v_scale[others] = float("inf")
    q = make_rows(2, heads * per * dim, dtype, cuda, 18)
    starts = _kv.starts_of([2], cuda)
    out = run_attention(cache, q, heads * per, starts, cuda)
    check_attention(cache, q, starts, out, heads * per)
    # the last token is NaN: its own row sees it, the row before does not
    before = out[0].clone()
    cache.tail_k[0, :, 35] = float("nan")
    cache.tail_v[0, :, 35] = float("inf")
    out = run_attention(cache, q, heads * per, starts, cuda)
    assert torch.equal(out[0], before) and bool(out[1].isnan().all())


def test_attention_nan_and_infinite_queries_stay_in_their_rows(cuda):
    heads, per, dim = 1, 4, 128
    cache = _kv.random_cache([300], heads, dim, torch.float32, cuda, seed=19)
    q = make_rows(3, heads * per * dim, torch.float32, cuda, 20)
    starts = _kv.starts_of([3], cuda)
    clean = run_attention(cache, q, heads * per, starts, cuda)
    q[1, 5] = float("nan")
    q[1, dim + 5] = float("inf")
    out = run_attention(cache, q, heads * per, starts, cuda)
    assert bool(out[1, :2 * dim].isnan().all())
    assert torch.equal(out[1, 2 * dim:], clean[1, 2 * dim:])
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,news", [([1], [1]), ([64, 65, 0, 300], [1, 1, 0, 1]), ([200, 90], [50, 90])])
def test_attention_weights(dtype, dim, lens, news, cuda):
    heads, per = 2, 3
    cache = _kv.random_cache(lens, heads, dim, dtype, cuda, seed=21, weights=True)
    q = make_rows(sum(news), heads * per * dim, dtype, cuda, 22)
    starts = _kv.starts_of(news, cuda)
    before = [_kv.seq_weights(cache, b).double() for b in range(len(lens))]
    w0, tw0 = cache.weight.clone(), cache.tail_weight.clone()
    out = run_attention(cache, q, heads * per, starts, cuda, accumulate=True)
    weights = check_attention(cache, q, starts, out, heads * per)
    touched = torch.zeros_like(cache.weight, dtype=torch.bool)
    for b, L in enumerate(lens):
        got = _kv.seq_weights(cache, b).double()
        want = before[b] + weights[b]
        # a sum of up to per * n terms p <= 1 in 32 bits, each p within 2^-12 (the bound of ``_kv.attention`` without the
        # rounding of p to fp16, which the sum of weights does not take: 2 ds + 2^-22 + sums < 2^-12 at these sizes)
        assert float((got - want).abs().max() if L else 0) <= per * max(news) * 2.0 ** -12
        assert float(((got - want).abs() - 2.0 ** -12 * weights[b] - 2.0 ** -23 * want).max() if L else 0) <= 0
        touched[cache.table[b, :L // PAGE].long()] = True
    assert torch.equal(cache.weight[~touched], w0[~touched])
    for b, L in enumerate(lens):
        assert torch.equal(cache.tail_weight[b, :, L % PAGE:], tw0[b, :, L % PAGE:])


def test_attention_of_sequences_that_share_pages(cuda):
    """A common prefix kept once: two sequences with the same first pages, weights of both added up."""
    heads, per, dim = 1, 2, 64
    cache = _kv.random_cache([200, 140], heads, dim, torch.float16, cuda, seed=23, weights=True)
    cache.table[1, :2] = cache.table[0, :2]
    w0 = cache.weight.clone().double().cpu()
    q = make_rows(2, heads * per * dim, torch.float16, cuda, 24)
    starts = _kv.starts_of([1, 1], cuda)
    out = run_attention(cache, q, heads * per, starts, cuda, accumulate=True)
    weights = check_attention(cache, q, starts, out, heads * per)
    page = int(cache.table[0, 0])
    want = w0[page, 0] + weights[0][0, :PAGE] + weights[1][0, :PAGE]
    assert float((cache.weight[page, 0].double().cpu() - want).abs().max()) <= 2.0 ** -10


# ---- eviction ----

def expected_eviction(cache, b, budget, sinks, recent):
    """The kept slots of sequence b per head, or None."""
    L = int(cache.lens[b])
    if L <= budget:
        return None
    kept = []
    for w in _kv.seq_weights(cache, b):
        order = torch.where(w.isnan(), -float("inf"), w).double()
        order[:sinks] = float("inf")
        order[L - recent:] = float("inf")
        # the earlier of equal ones first
        idx = sorted(range(L), key=lambda i: (not (i < sinks or i >= L - recent), -float(order[i]), i))[:budget]
        kept.append(sorted(idx))
    return kept


def check_eviction(cache, budget, sinks, recent, device):
    seqs, heads = cache.table.shape[0], cache.k.shape[1]
    nb = budget // PAGE
    used = set(cache.table[cache.table >= 0].tolist())
    free = [p for p in range(cache.k.shape[0]) if p not in used]
    spare = torch.tensor(free[:seqs * nb], dtype=torch.int32, device=device).view(seqs, nb)
    plans = [expected_eviction(cache, b, budget, sinks, recent) for b in range(seqs)]
    ks = [_kv.sequence(cache, b, "k") for b in range(seqs)]
    vs = [_kv.sequence(cache, b, "v") for b in range(seqs)]
    ws = [_kv.seq_weights(cache, b) for b in range(seqs)]
    table0, spare0, lens0 = cache.table.clone(), spare.clone(), cache.lens.clone()
    tails = [t.clone() for t in (cache.tail_k, cache.tail_v, cache.tail_weight)]
    ops.kv_evict(cache, spare, budget, sinks=sinks, recent=recent)
    wait(device)
    for b, plan in enumerate(plans):
        if plan is None:
            assert torch.equal(cache.table[b], table0[b]) and torch.equal(spare[b], spare0[b])
            assert int(cache.lens[b]) == int(lens0[b])
            assert torch.equal(_kv.sequence(cache, b, "k"), ks[b]) and torch.equal(_kv.seq_weights(cache, b).view(torch.int32), ws[b].view(torch.int32))
            continue
        assert int(cache.lens[b]) == budget
        assert torch.equal(cache.table[b, :nb], spare0[b]) and torch.equal(spare[b], table0[b, :nb])
        assert torch.equal(cache.table[b, nb:], table0[b, nb:])
        for h in range(heads):
            for j in range(nb):
                page, slots = int(cache.table[b, j]), plan[h][j * PAGE:(j + 1) * PAGE]
                for name, x in (("k", ks[b]), ("v", vs[b])):
                    codes, scale = _kv.quantised(x[slots, h])
                    assert torch.equal(getattr(cache, name + "_scale")[page, h].cpu(), scale), (name, b, h, j)
                    assert torch.equal(getattr(cache, name)[page, h].cpu(), codes), (name, b, h, j)
                assert torch.equal(cache.weight[page, h].cpu().view(torch.int32), ws[b][h, slots].view(torch.int32))
    for t, was in zip((cache.tail_k, cache.tail_v, cache.tail_weight), tails):
        assert torch.equal(t, was)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,budget,sinks,recent", [
    ([65], 64, 0, 0),
    ([200, 64, 63, 0], 64, 4, 20),
    ([300, 129, 128], 128, 0, 128),
    ([400, 193], 192, 100, 92),
    ([2500, 1100], 1024, 4, 64),
])
def test_evict(dtype, dim, lens, budget, sinks, recent, cuda):
    cache = _kv.random_cache(lens, 2, dim, dtype, cuda, seed=25, weights=True, extra=len(lens) * budget // PAGE,
                             width=max(max(lens) // PAGE + 1, budget // PAGE))
    check_eviction(cache, budget, sinks, recent, cuda)


def test_evict_ties_and_odd_weights(cuda):
    """Weights that are all equal, zero of both signs, negative, infinite, NaN, and the smallest above zero."""
    cache = _kv.random_cache([500, 500, 500], 2, 64, torch.bfloat16, cuda, seed=26, weights=True, extra=9)
    cache.weight.zero_()
    cache.tail_weight.zero_()
    pages = cache.table[1, :7].long()
    cache.weight[pages[2], 0, 10:20] = -0.0
    cache.weight[pages[3], 0, 5:50] = -1.0
    cache.weight[pages[4], 0, :40] = 1e-45
    cache.weight[pages[5], 1, 3] = float("inf")
    cache.weight[pages[5], 1, 4] = float("nan")
    cache.weight[pages[0], 1, :60] = float("nan")
    # few different values: the border falls among equal ones
    cache.weight[cache.table[2, :7].long()] = torch.randint(0, 3, (7, 2, PAGE), generator=torch.Generator().manual_seed(27)).float().to(cuda)
    check_eviction(cache, 192, 3, 10, cuda)


def test_evict_again_uses_the_old_pages(cuda):
    """Two evictions in a row, with tokens in between, need no other pages than the two sets."""
    heads, dim, budget = 2, 64, 128
    cache = _kv.random_cache([300], heads, dim, torch.float16, cuda, seed=28, weights=True, extra=8, width=6)
    used = set(cache.table[0, :4].tolist())
    free = [p for p in range(cache.k.shape[0]) if p not in used]
    cache.table[0, 4:] = torch.tensor(free[:2], dtype=torch.int32, device=cuda)
    spare = torch.tensor([free[2:4]], dtype=torch.int32, device=cuda)
    every = sorted(cache.table[0].tolist() + spare[0].tolist())
    for step in range(3):
        ops.kv_evict(cache, spare, budget, sinks=4, recent=32)
        wait(cuda)
        assert int(cache.lens[0]) == budget and sorted(cache.table[0].tolist() + spare[0].tolist()) == every
        x = make_rows(100, heads * dim, torch.float16, cuda, 29 + step)
        fill(cache, [100], x, x, dim, cuda)
        wait(cuda)
        check_tail = cache.tail_k[0, :, :100 - PAGE].transpose(0, 1).reshape(-1, heads * dim)
        assert torch.equal(check_tail, x[PAGE:])


# ---- index errors ----

def test_bad_pages_and_lengths_are_reported(cuda):
    heads, per, dim = 1, 2, 64
    cache = _kv.random_cache([200, 100], heads, dim, torch.float16, cuda, seed=30, weights=True, extra=8)
    q = make_rows(2, heads * per * dim, torch.float16, cuda, 31)
    starts = _kv.starts_of([1, 1], cuda)
    good = run_attention(cache, q, heads * per, starts, cuda)
    page = int(cache.table[0, 1])
    for bad in (-1, cache.k.shape[0], 1 << 30):
        cache.table[0, 1] = bad
        out = torch.full_like(good, 7.0)
        ops.attention_cached(_kv.rows(q, heads * per, dim), cache, starts, out, accumulate=True)
        with pytest.raises(native.H3Error, match="page id"):
            wait(cuda)
        assert torch.equal(out[1], good[1]) and not torch.equal(out[0], good[0])
        before = [t.clone() for t in (cache.k, cache.v, cache.weight)]
        spare = torch.tensor([[5], [6]], dtype=torch.int32, device=cuda)
        ops.kv_evict(cache, spare, PAGE, sinks=4, recent=10)
        with pytest.raises(native.H3Error, match="page id"):
            wait(cuda)
        assert cache.lens.tolist()[0] == 200 and spare[0, 0] == 5
        for t, was in zip((cache.k, cache.v, cache.weight), before):
            t.copy_(was)
        cache.lens.copy_(torch.tensor([200, 100]))
        cache.table[1, 0] = int(spare[1, 0]) if int(cache.table[1, 0]) == 6 else cache.table[1, 0]
    cache.table[0, 1] = page
    cache.lens[0] = 64 * cache.table.shape[1] + 64
    for call in (lambda: ops.attention_cached(_kv.rows(q, heads * per, dim), cache, starts, torch.empty_like(good)),
                 lambda: ops.kv_append(cache, _kv.rows(q, 1, dim), _kv.rows(q, 1, dim), starts),
                 lambda: ops.kv_evict(cache, torch.tensor([[5], [6]], dtype=torch.int32, device=cuda), PAGE, recent=8)):
        call()
        with pytest.raises(native.H3Error, match="lengths"):
            wait(cuda)
    cache.lens.copy_(torch.tensor([200, 100]))
    for s in ([0, 1, 9], [-1, 1, 2], [1, 0, 2]):
        bad = torch.tensor(s, dtype=torch.int32, device=cuda)
        ops.attention_cached(_kv.rows(q, heads * per, dim), cache, bad, torch.empty_like(good))
        with pytest.raises(native.H3Error, match="starts"):
            wait(cuda)
    wait(cuda)
    assert torch.equal(run_attention(cache, q, heads * per, starts, cuda)[0], good[0])


# ---- many query rows (tcgen05 for 16-bit types) ----

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,per,lens,news", [
    (1, 4, [64], [64]),                     # one page, one tile
    (2, 4, [200], [200]),                   # a whole prompt: pages and a tail
    (1, 1, [300], [256]),
    (1, 3, [700, 130, 0, 64], [300, 7, 0, 60]),   # rows of a token over a tile's edge; short sequences beside a long one
    (1, 8, [1000], [130]),                  # several tiles
    (1, 16, [63], [63]),                    # the tail alone
    (1, 2, [100, 5], [200, 90]),            # more rows than tokens: the first ones see nothing
    (2, 2, [2500], [64]),                   # few tiles: the keys are split
])
def test_attention_of_many_rows(dtype, dim, heads, per, lens, news, cuda):
    cache = _kv.random_cache(lens, heads, dim, dtype, cuda, seed=len(lens) + dim + 40)
    q = make_rows(sum(news), heads * per * dim, dtype, cuda, 41)
    starts = _kv.starts_of(news, cuda)
    out = run_attention(cache, q, heads * per, starts, cuda)
    check_attention(cache, q, starts, out, heads * per)


@pytest.mark.parametrize("dtype", TYPES)
def test_many_rows_with_few_tiles_in_the_grid(dtype, cuda):
    """A hint of 128 new tokens for a sequence that brings 1,100: a CTA takes several tiles one after the other."""
    cache = _kv.random_cache([1200, 600], 1, 64, dtype, cuda, seed=42)
    q = make_rows(1100 + 130, 2 * 64, dtype, cuda, 43)
    starts = _kv.starts_of([1100, 130], cuda)
    out = run_attention(cache, q, 2, starts, cuda, max_new=128)
    check_attention(cache, q, starts, out, 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,news", [([150], [150]), ([900], [64])])
def test_many_rows_value_scales_of_many_sizes(dtype, lens, news, cuda):
    """Pages whose value scales differ by factors of 2^20, and some that are 0: every page counts by its own."""
    cache = _kv.random_cache(lens, 1, 64, dtype, cuda, seed=44, weights=True)
    pages = cache.table[0, :lens[0] // PAGE].long()
    for i, p in enumerate(pages):
        cache.v_scale[p] = 0.02 * 2.0 ** (-20 if i % 3 == 1 else 0)
        if i % 3 == 2:
            cache.v_scale[p] = 0
            cache.v[p] = 0
    q = make_rows(news[0], 4 * 64, dtype, cuda, 45)
    starts = _kv.starts_of(news, cuda)
    before = _kv.seq_weights(cache, 0).double()
    out = run_attention(cache, q, 4, starts, cuda, accumulate=True)
    weights = check_attention(cache, q, starts, out, 4)
    got = _kv.seq_weights(cache, 0).double()
    assert float(((got - before - weights[0]).abs() - 2.0 ** -12 * weights[0] - 2.0 ** -23 * (before + weights[0])).max()) <= 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_rows_hidden_slots_may_hold_anything(dtype, cuda):
    """NaN and infinities behind the end, in later tokens, in other sequences' pages and in other rows of q."""
    n, per, dim = 100, 2, 64
    cache = _kv.random_cache([n], 1, dim, dtype, cuda, seed=46)
    others = [p for p in range(cache.k.shape[0]) if p != int(cache.table[0, 0])]
    cache.k_scale[others] = float("nan")
    cache.v_scale[others] = float("inf")
    cache.tail_k[0, :, n - PAGE:] = float("nan")
    cache.tail_v[0, :, n - PAGE:] = float("inf")
    q = make_rows(n, per * dim, dtype, cuda, 47)
    starts = _kv.starts_of([n], cuda)
    clean = run_attention(cache, q, per, starts, cuda)
    check_attention(cache, q, starts, clean, per)
    at = 90 - PAGE
    cache.tail_v[0, 0, at, 5] = float("inf")
    cache.tail_v[0, 0, at + 2, 6] = float("nan")
    out = run_attention(cache, q, per, starts, cuda).view(n, per, dim)
    was = clean.view(n, per, dim)
    assert torch.equal(out[:90], was[:90]) and torch.equal(out[:, :, 7:], was[:, :, 7:])
    assert bool((out[90:, :, 5] == float("inf")).all()) and bool(out[92:, :, 6].isnan().all())
    assert torch.equal(out[90:92, :, 6], was[90:92, :, 6])
    cache.tail_k[0, 0, at, 3] = float("nan")
    q[7, 1], q[8, dim + 1] = float("nan"), float("inf")
    out = run_attention(cache, q, per, starts, cuda).view(n, per, dim)
    bad = torch.zeros(n, per, dtype=torch.bool, device=cuda)
    bad[90:] = bad[7, 0] = bad[8, 1] = True
    assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], was[~bad])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,per,L", [(75, 1, 75), (50, 3, 1500)])
def test_many_rows_of_a_warp_that_see_unlike_tails(dtype, dim, n, per, L, cuda):
    """A tile that ends inside a warp, and infinities in every 32 features of the tail that some rows of a warp see and others
    do not: every feature of every row comes out as if it were alone. Once in one piece, once with the keys split."""
    cache = _kv.random_cache([L], 1, dim, dtype, cuda, seed=49)
    q = make_rows(n, per * dim, dtype, cuda, 50)
    starts = _kv.starts_of([n], cuda)
    clean = run_attention(cache, q, per, starts, cuda)
    check_attention(cache, q, starts, clean, per)
    tail = L % PAGE
    want = clean.view(n, per, dim).clone()
    for i in range(min(tail, n)):                  # tail row tail - 1 - i is seen by the last i + 1 tokens
        if i % 3 == 0:
            feature = (7 * i + 32 * (i // 3)) % dim
            sign = float("inf") if i % 2 else -float("inf")
            if cache.tail_v[0, 0, :tail, feature].isfinite().all():
                cache.tail_v[0, 0, tail - 1 - i, feature] = sign
                want[n - 1 - i:, :, feature] = sign
    out = run_attention(cache, q, per, starts, cuda)
    # what is finite: the tail's power of two may have moved with the values that became infinite
    infinite = ~want.isfinite()
    out = out.view(n, per, dim)
    assert torch.equal(out[infinite], want[infinite])
    cache.tail_v[0, 0, :tail][~cache.tail_v[0, 0, :tail].isfinite()] = 0
    exact, _, bound = _kv.attention(cache, q, per, starts)
    off = ((out.double().cpu() - exact.view(n, per, dim)).abs() - bound.view(n, per, dim))[~infinite.cpu()]
    assert float(off.max()) <= 0, f"off by {float(off.max()):.3g} more than the roundings"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("seqs,heads,max_len", [(40, 2, 64), (33, 1, 1), (700, 8, None)])
def test_attention_of_many_sequences_in_whole_pieces(dtype, seqs, heads, max_len, cuda):
    """More sequences than a warp has lanes, and no unit cut: by a hint of short lengths, or because there are many units."""
    g = torch.Generator().manual_seed(seqs)
    lens = torch.randint(0, 300, (seqs,), generator=g).tolist()
    news = [0 if b % 9 == 4 else 1 for b in range(seqs)]
    cache = _kv.random_cache(lens, heads, 64, dtype, cuda, seed=seqs)
    q = make_rows(sum(news), heads * 2 * 64, dtype, cuda, 51)
    starts = _kv.starts_of(news, cuda)
    out = run_attention(cache, q, heads * 2, starts, cuda, max_new=1, max_len=max_len)
    check_attention(cache, q, starts, out, heads * 2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("low", [0, 1])
def test_many_rows_whose_reference_moves_between_halves(dtype, low, cuda):
    """The second half of a key tile is taken first; keys of the first whose scores are some 2^8.5 to 2^12 times as large move
    the reference of the weights taken before. Only those have values, so that their roundings alone are seen: one for
    each weight. ``low``: the same with the move between two key tiles."""
    n, pages = 4096, 5
    cache = _kv.random_cache([64 * pages + n], 1, 64, dtype, cuda, seed=52)
    cache.k.zero_()
    cache.v.zero_()
    cache.k_scale.fill_(0.05)
    cache.v_scale.fill_(2000.0)
    page = cache.table[0, :pages + n // PAGE].long()
    for i in range(len(page)):
        cache.k[page[i], 0, :, :2] = -60
    first, second = (0, 1) if not low else (2, 1)      # `first` is read after `second` and scores higher
    cache.k[page[first], 0, :, :2] = 60
    cache.k[page[second], 0, :, :2] = -5
    cache.k[page[second], 0, 0, :2] = 0                # the largest of its half, with no value
    cache.v[page[second], 0, 1:, :] = 100
    g = torch.Generator().manual_seed(53)
    q = torch.zeros(n, 64)
    q[:, 0] = (0.1417 + 0.0583 * torch.rand(n, generator=g)) * 8 / (0.05 * 1.4427)
    q[:, 1] = 0.05 * torch.rand(n, generator=g)        # scores finer than the first feature's steps
    q = q.to(dtype).to(cuda)
    starts = _kv.starts_of([n], cuda)
    out = run_attention(cache, q, 1, starts, cuda)
    check_attention(cache, q, starts, out, 1)


def test_a_wait_that_gave_up_and_a_bad_page_are_both_reported(cuda):
    cache = _kv.random_cache([200], 1, 64, torch.float16, cuda, seed=54)
    q = make_rows(1, 64, torch.float16, cuda, 55)
    starts = _kv.starts_of([1], cuda)
    cache.table[0, 1] = -1
    ctx = ops.context(cuda)
    ops.attention_cached(_kv.rows(q, 1, 64), cache, starts, torch.empty_like(q))
    ctx.selftest_wait_timeout(2_000_000)               # 2 ms
    with pytest.raises(native.H3Error, match="gave up.*page id"):
        ctx.wait()
    ctx.wait()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("L,n,per", [(100, 1, 1), (100, 3, 4), (4000, 2, 3), (130, 66, 2), (4000, 64, 1), (60, 60, 1)])
def test_infinite_values_of_small_weights(dtype, dim, L, n, per, cuda):
    """An infinite value in the tail whose key's score lies so far below the others that its weight is 0 in 32 bits: its
    feature is infinite in the rows that see it, NaN where both signs meet or a value is NaN, on every path and through
    every join; the other features stay."""
    cache = _kv.random_cache([L], 1, dim, dtype, cuda, seed=56)
    q = make_rows(n, per * dim, dtype, cuda, 57)
    q[:, ::dim] = 8                                    # feature 0 of every head
    tail = L % PAGE
    seen = (max(tail - 3, 0), max(tail - 2, 1))        # two keys that the last rows see
    cache.tail_k[0, 0, seen[0]:seen[1] + 1] = 0
    cache.tail_k[0, 0, seen[0]:seen[1] + 1, 0] = -4000.0
    starts = _kv.starts_of([n], cuda)
    clean = run_attention(cache, q, per, starts, cuda).view(n, per, dim)
    check_attention(cache, q, starts, clean.view(n, -1), per)
    inf = float("inf")
    cache.tail_v[0, 0, seen[0], 5] = inf
    cache.tail_v[0, 0, seen[1], 9] = -inf
    cache.tail_v[0, 0, seen[0], 40], cache.tail_v[0, 0, seen[1], 40] = inf, -inf
    cache.tail_v[0, 0, seen[1], dim - 1] = float("nan")
    out = run_attention(cache, q, per, starts, cuda).view(n, per, dim)
    pos = torch.arange(L - n, L) - (L - tail)
    sees0, sees1 = pos >= seen[0], pos >= seen[1]
    assert bool(sees1.any())
    want = clean.clone()
    want[sees0.to(cuda), :, 5] = inf
    want[sees1.to(cuda), :, 9] = -inf
    want[sees0.to(cuda), :, 40] = inf
    want[sees1.to(cuda), :, 40] = float("nan")
    want[sees1.to(cuda), :, dim - 1] = float("nan")
    odd = ~want.isfinite()
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.nan_to_num(7.0, 1e4, -1e4)[odd], want.nan_to_num(7.0, 1e4, -1e4)[odd])
    for t, f in ((seen[0], 5), (seen[1], 9), (seen[0], 40), (seen[1], 40), (seen[1], dim - 1)):
        cache.tail_v[0, 0, t, f] = 0
    exact, _, bound = _kv.attention(cache, q, per, starts)
    off = ((out.double().cpu() - exact.view(n, per, dim)).abs() - bound.view(n, per, dim))[~odd.cpu()]
    assert float(off.max()) <= 0


@pytest.mark.parametrize("max_new", [12, 64, 1000, None])
def test_a_hint_below_the_rows_of_a_call_takes_no_more_memory(max_new, cuda):
    """The partial results of 100,000 rows with a hint of a few: as many as there are without it (30 GB before)."""
    cache = ops.KVCache.empty(1, 1, 4096, 8, 128, torch.float16, cuda)
    nbytes = ops.context(cuda).attention_cached_work(cache._ptr, 100000, 32, max_new or 0, 0, 0)
    assert nbytes <= 2 * 148 * 256 * 130 * 4


@pytest.mark.parametrize("max_new", [1, 64, 100, 1 << 40])
def test_append_hints_only_divide_the_work(max_new, cuda):
    heads, dim, news = 2, 64, [700, 3, 130]
    k, v = make_rows(sum(news), heads * dim, torch.bfloat16, cuda, 58), make_rows(sum(news), heads * dim, torch.bfloat16, cuda, 59)
    cache = ops.KVCache.empty(36, 3, 11, heads, dim, torch.bfloat16, cuda)
    scatter_table(cache, cuda)
    cache.lens.copy_(torch.tensor(news, dtype=torch.int32))
    ops.kv_append(cache, _kv.rows(k, heads, dim), _kv.rows(v, heads, dim), _kv.starts_of(news, cuda), max_new=max_new)
    wait(cuda)
    at = 0
    for b, n in enumerate(news):
        check_written(cache, b, heads, k[at:at + n].view(n, heads, dim), v[at:at + n].view(n, heads, dim))
        at += n


def test_evict_from_more_tokens_than_shared_memory_holds_keys_of(cuda):
    cache = _kv.random_cache([50001, 300], 1, 64, torch.float16, cuda, seed=60, weights=True, extra=10)
    cache.weight.mul_(16).floor_()                     # many equal ones
    check_eviction(cache, 256, 4, 40, cuda)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("stale", [-(1 << 31), 0, 77])
def test_evict_does_not_go_by_what_work_held(dtype, stale, cuda):
    """The same eviction with a work memory full of each of: what stands for a sequence that is left alone, and places of
    other tokens. Its kernels are launched while the one before still runs: none may read work before that one has ended."""
    heads, dim, budget, lens = 2, 64, 2 * PAGE, [129, 3000, 100, 700]
    cache = _kv.random_cache(lens, heads, dim, dtype, cuda, seed=61, weights=True, extra=8)
    used = set(cache.table[cache.table >= 0].tolist())
    spare = torch.tensor([p for p in range(cache.k.shape[0]) if p not in used][:8], dtype=torch.int32, device=cuda).view(4, 2)
    start = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.weight, cache.table, cache.lens, spare)]
    work = torch.empty(4 * heads * budget, dtype=torch.int32, device=cuda)
    plans = [expected_eviction(cache, b, budget, 4, 16) for b in range(4)]
    before = [_kv.sequence(cache, b, "k") for b in range(4)]
    weights = [_kv.seq_weights(cache, b) for b in range(4)]
    for _ in range(40):
        for t, was in zip((cache.k, cache.v, cache.k_scale, cache.v_scale, cache.weight, cache.table, cache.lens, spare), start):
            t.copy_(was)
        work.fill_(stale)
        ops.context(cuda).kv_evict(cache._ptr, spare.data_ptr(), budget, 4, 16, work.data_ptr(), work.numel() * 4)
        wait(cuda)
        assert cache.lens.tolist() == [128, 128, 100, 128]
        for b, plan in enumerate(plans):
            if plan is None:
                continue
            w = _kv.seq_weights(cache, b)
            for h in range(heads):
                assert torch.equal(w[h], weights[b][h, plan[h]])
                for j in range(2):
                    page = int(cache.table[b, j])
                    codes, scale = _kv.quantised(before[b][plan[h][j * PAGE:(j + 1) * PAGE], h])
                    assert torch.equal(cache.k[page, h].cpu(), codes) and torch.equal(cache.k_scale[page, h].cpu(), scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,per,lens,news", [(8, 4, [9000], [1]), (4, 4, [3000, 70, 900] * 12, [1, 0, 1] * 12), (2, 4, [3000], [100]),
                                                 (2, 4, [5000, 300], [5, 3])])
def test_attention_does_not_go_by_what_work_held(dtype, heads, per, lens, news, cuda):
    """The same bits whatever the work memory holds before the call, and the definition's values: pieces and splits that are
    joined, and weights, by kernels that are launched while the one before still runs."""
    cache = _kv.random_cache(lens, heads, 64, dtype, cuda, seed=62, weights=True)
    q = make_rows(sum(news), heads * per * 64, dtype, cuda, 63)
    starts = _kv.starts_of(news, cuda)
    w0, t0 = cache.weight.clone(), cache.tail_weight.clone()
    ctx, rows, first = ops.context(cuda), _kv.rows(q, heads * per, 64), None
    nbytes = ctx.attention_cached_work(cache._ptr, sum(news), heads * per, max(news), max(lens), 1)
    assert nbytes > 16 * sum(news) * heads * per           # there are partial results
    work = torch.empty((nbytes + 15) // 16 * 4, device=cuda)
    for held in (float("nan"), 0.0, float("inf"), -3e38, 1.4e-45) * 4:
        work.fill_(held)
        cache.weight.copy_(w0)
        cache.tail_weight.copy_(t0)
        out = torch.full_like(q, 7.0)
        ctx.attention_cached(cache._ptr, rows.ptr(), sum(news), heads * per, rows.stride, starts.data_ptr(), max(news), max(lens),
                             out.data_ptr(), 1, work.data_ptr(), nbytes)
        wait(cuda)
        if first is None:
            check_attention(cache, q, starts, out, heads * per)
            first = out, cache.weight.clone(), cache.tail_weight.clone()
        for a, b in zip(first, (out, cache.weight, cache.tail_weight)):
            assert torch.equal(a, b)
