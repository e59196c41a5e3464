"""The text model's operators as a step uses them: linear layer, norm and rotation, append, attention, linear layer, eviction;
every result against its definition in 64 bits from the inputs that the step gave it, and the same steps captured, replayed
and beside each other bit for bit. Also the ranges that only large calls reach."""
import pytest
import torch

import _kv
import test_gpu_int4_linear as lin4
from _kv import PAGE
from sycl_minimax_h3_b200 import native, ops
from test_gpu_kvcache import check_attention, check_eviction, check_written, make_rows, scatter_table

pytestmark = pytest.mark.gpu

HEADS, PER, DIM, WIDTH, GROUP = 2, 3, 64, 256, 64
HQ = HEADS * PER


def wait(device):
    ops.context(device).wait()


class Layer:
    def __init__(self, dtype, device):
        n = (HQ + 2 * HEADS) * DIM
        self.qkv = lin4.make(1, n, WIDTH, GROUP, dtype, torch.float32, True, True, device, seed=1)
        self.out = lin4.make(1, WIDTH, HQ * DIM, 0, dtype, dtype, False, False, device, seed=2)
        self.norm = torch.linspace(0.5, 1.5, DIM, device=device)
        angle = torch.arange(4096, device=device)[:, None] * 10000.0 ** (-torch.arange(0, DIM, 2, device=device) / DIM)
        self.cs = torch.stack((angle.cos(), angle.sin()), -1).contiguous()

    def parts(self, qkv):
        w = qkv.shape[1]
        return (ops.Rows(qkv, 0, w, qkv.shape[0], HQ, DIM), ops.Rows(qkv, HQ * DIM, w, qkv.shape[0], HEADS, DIM),
                ops.Rows(qkv, (HQ + HEADS) * DIM, w, qkv.shape[0], HEADS, DIM))

    def rows(self, x, qkv, at):
        self.qkv[5].forward(x, qkv)
        q, k, v = self.parts(qkv)
        cs = self.cs.index_select(0, at)
        ops.rms_rope(q, self.norm, 1e-6, cs, DIM)
        ops.rms_rope(k, self.norm, 1e-6, cs, DIM)
        return q, k, v

    def step(self, x, at, cache, starts, spare, budget, qkv, mid, y, **hints):
        q, k, v = self.rows(x, qkv, at)
        ops.kv_append(cache, k, v, starts)
        ops.attention_cached(q, cache, starts, mid, accumulate=True, **hints)
        self.out[5].forward(mid, y)
        ops.kv_evict(cache, spare, budget, sinks=4, recent=16)


def new_cache(dtype, device, seqs=3, width=6):
    cache = ops.KVCache.empty(seqs * width + 2 * seqs, seqs, width, HEADS, DIM, dtype, device, True)
    scatter_table(cache, device)
    used = set(cache.table.flatten().tolist())
    spare = torch.tensor([p for p in range(cache.k.shape[0]) if p not in used][:2 * seqs], dtype=torch.int32, device=device)
    return cache, spare.view(seqs, 2)


@pytest.mark.parametrize("dtype", lin4.TYPES)
def test_steps_of_a_layer(dtype, cuda):
    """Prompts of unequal lengths, single tokens over a page's end, and an eviction; each operator on what the one before left."""
    layer, (cache, _) = Layer(dtype, cuda), new_cache(dtype, cuda)
    seen = [torch.zeros(0, HEADS, DIM, dtype=dtype)] * 3, [torch.zeros(0, HEADS, DIM, dtype=dtype)] * 3
    for step, news in enumerate(([150, 63, 1], [1, 1, 0], [1, 1, 1], [40, 1, 70], [1, 1, 1])):
        T, old = sum(news), cache.lens.tolist()
        x = make_rows(T, WIDTH, dtype, cuda, step)
        at = torch.cat([torch.arange(l, l + n) for l, n in zip(old, news)]).to(cuda)
        starts = _kv.starts_of(news, cuda)
        qkv = torch.empty(T, (HQ + 2 * HEADS) * DIM, dtype=dtype, device=cuda)
        codes, scale, z, b, _, lin = layer.qkv
        lin.forward(x, qkv)
        wait(cuda)
        lin4.check(codes, scale, z, b, x.cpu(), GROUP, qkv)
        q, k, v = layer.rows(x, qkv, at)
        cache.lens.add_(torch.tensor(news, dtype=torch.int32, device=cuda))
        ops.kv_append(cache, k, v, starts)
        mid = torch.empty(T, HQ * DIM, dtype=dtype, device=cuda)
        wait(cuda)
        before = [_kv.seq_weights(cache, i).double() for i in range(3)]
        ops.attention_cached(q, cache, starts, mid, accumulate=True)
        wait(cuda)
        rows = qkv.cpu().view(T, -1, DIM)
        for i in range(3):
            for which, first in ((0, HQ), (1, HQ + HEADS)):
                seen[which][i] = torch.cat((seen[which][i], rows[int(starts[i]):int(starts[i + 1]), first:first + HEADS]))
            check_written(cache, i, HEADS, seen[0][i], seen[1][i])
        weights = check_attention(cache, qkv[:, :HQ * DIM].contiguous(), starts, mid, HQ)
        # a weight is off by twice the error of a score, (dim + 8) 2^-23 sum |q k| / sqrt(dim) < 72 2^-23 64 1.5^2 / 8, and the
        # rounding of the p that its row's sum is made of, 2^-11: less than 2^-9 of itself; then the sum's own rounding
        for i in range(3):
            was = torch.zeros_like(weights[i])
            was[:, :before[i].shape[1]] = before[i]
            got = _kv.seq_weights(cache, i).double()
            assert bool(((got - was - weights[i]).abs() <= 2.0 ** -9 * weights[i] + 2.0 ** -22 * (was + weights[i])).all())
        y = torch.empty(T, WIDTH, dtype=dtype, device=cuda)
        codes, scale, z, b, _, lin = layer.out
        lin.forward(mid, y)
        wait(cuda)
        lin4.check(codes, scale, z, b, mid.cpu(), 0, y)
    check_eviction(cache, 2 * PAGE, 4, 16, cuda)
    assert cache.lens.tolist() == [128, 67, 73]


def run(layer, dtype, device, steps, between):
    """`steps` single tokens of three sequences from lens 100, 60, 0 on; between(step) runs a prepared step."""
    g = torch.Generator().manual_seed(9)
    xs = torch.randn(steps, 3, WIDTH, generator=g).to(dtype).to(device)
    cache, spare = new_cache(dtype, device)
    cache.k.copy_(torch.randint(-127, 128, cache.k.shape, generator=g))
    cache.v.copy_(torch.randint(-127, 128, cache.v.shape, generator=g))
    cache.k_scale.fill_(0.02)
    cache.v_scale.fill_(0.01)
    cache.lens.copy_(torch.tensor([100, 60, 0]))
    at = torch.tensor([100, 60, 0], device=device)
    x, y = torch.empty(3, WIDTH, dtype=dtype, device=device), torch.empty(3, WIDTH, dtype=dtype, device=device)
    qkv = torch.empty(3, (HQ + 2 * HEADS) * DIM, dtype=dtype, device=device)
    mid = torch.empty(3, HQ * DIM, dtype=dtype, device=device)
    starts = _kv.starts_of([1, 1, 1], device)
    ys = torch.empty(steps, 3, WIDTH, dtype=dtype, device=device)

    def step():
        cache.lens.add_(1)
        layer.step(x, at, cache, starts, spare, 2 * PAGE, qkv, mid, y, max_new=1, max_len=4096)
        at.add_(1)

    go = between(step)
    for i in range(steps):
        x.copy_(xs[i])
        go()
        ys[i].copy_(y)
    return ys, cache, spare


def parts(r):
    return [r[0], r[2]] + [t for t in (r[1].k, r[1].v, r[1].k_scale, r[1].v_scale, r[1].tail_k, r[1].tail_v, r[1].table, r[1].lens,
                                       r[1].weight, r[1].tail_weight)]


@pytest.mark.parametrize("dtype", lin4.TYPES)
def test_a_captured_step_and_steps_on_two_streams_give_the_same_bits(dtype, cuda):
    """90 tokens: over pages' ends and evictions from 128 on. The first use of a stream may be a capture; two runs on two
    streams do not disturb each other."""
    layer = Layer(dtype, cuda)
    eager = run(layer, dtype, cuda, 90, lambda step: step)
    wait(cuda)
    assert eager[1].lens.tolist() == [128, 128, 90]
    side, graphs = [torch.cuda.Stream(cuda) for _ in range(2)], []

    def captured(step):
        graphs.append(torch.cuda.CUDAGraph())
        stream = torch.cuda.current_stream(cuda)
        stream.synchronize()
        with torch.cuda.graph(graphs[-1], stream=stream):
            step()
        return graphs[-1].replay

    runs = []
    for s, how in zip(side, (captured, lambda step: step)):
        s.wait_stream(torch.cuda.current_stream(cuda))
        with torch.cuda.stream(s):
            runs.append(run(layer, dtype, cuda, 90, how))
    for s in side:
        with torch.cuda.stream(s):
            wait(cuda)
    for r in runs:
        for a, b in zip(parts(r), parts(eager)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_a_pool_of_more_than_four_gigabytes(cuda):
    """Pages whose codes lie past 2^31 and 2^32 bytes, rows whose elements do."""
    heads, per, dim, pages, stride = 8, 2, 128, 70000, 40_000_000
    lens, news = [300, 130], [66, 2]
    small = _kv.random_cache(lens, heads, dim, torch.bfloat16, cuda, seed=3, weights=True)
    big = ops.KVCache(*(torch.empty((pages,) + tuple(t.shape[1:]), dtype=t.dtype, device=cuda) for t in (small.k, small.v, small.k_scale, small.v_scale)),
                      small.tail_k, small.tail_v, small.table.clone(), small.lens, torch.empty(pages, heads, PAGE, device=cuda), small.tail_weight)
    far = torch.tensor([pages - 1 - 4001 * i for i in range(small.k.shape[0])], device=cuda)
    for name in ("k", "v", "k_scale", "v_scale", "weight"):
        getattr(big, name)[far] = getattr(small, name)
    big.table.copy_(torch.where(small.table >= 0, far[small.table.clamp(min=0).long()], -1))
    assert far.min() * heads * PAGE * dim > 1 << 31
    rows = torch.empty(sum(news), stride, dtype=torch.bfloat16, device=cuda)   # the last row starts past 2^31 elements
    width = (per + 2) * heads * dim
    rows[:, :width] = make_rows(sum(news), width, torch.bfloat16, cuda, 4)
    starts = _kv.starts_of(news, cuda)
    q = ops.Rows(rows, 0, stride, sum(news), heads * per, dim)
    k, v = (ops.Rows(rows, (per + i) * heads * dim, stride, sum(news), heads, dim) for i in range(2))
    ops.kv_append(big, k, v, starts)
    for few in (False, True):
        s = _kv.starts_of([1, 1], cuda) if few else starts
        out = torch.empty(2 if few else sum(news), heads * per * dim, dtype=torch.bfloat16, device=cuda)
        ops.attention_cached(ops.Rows(rows, 66 * stride, stride, 2, heads * per, dim) if few else q, big, s, out, accumulate=True)
        wait(cuda)
        check_attention(big, (rows[66:] if few else rows)[:, :heads * per * dim].contiguous(), s, out, heads * per)
    free = [int(p) for p in far if int(p) not in set(big.table.flatten().tolist())][:2] + [pages - 2, pages - 3]
    before = [_kv.sequence(big, b, "k") for b in range(2)], [_kv.seq_weights(big, b) for b in range(2)]
    spare = torch.tensor(free[:4], dtype=torch.int32, device=cuda).view(2, 2)
    ops.kv_evict(big, spare, 2 * PAGE, sinks=4, recent=124)
    wait(cuda)
    assert big.lens.tolist() == [128, 128]
    for b in range(2):                                     # nothing to choose: the first four and the last 124
        at = list(range(4)) + list(range(lens[b] - 124, lens[b]))
        assert torch.equal(_kv.seq_weights(big, b), before[1][b][:, at])
        for j in range(2):
            codes, scale = _kv.quantised(before[0][b][at[j * PAGE:(j + 1) * PAGE], heads - 1])
            page = int(big.table[b, j])
            assert torch.equal(big.k[page, heads - 1].cpu(), codes) and torch.equal(big.k_scale[page, heads - 1].cpu(), scale)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("per", [1, 40])
def test_starts_that_run_backwards_are_reported(dtype, per, cuda):
    """Row ranges that overlap stand for more pieces than the call has rows: reported, and the rest of the cache is whole."""
    heads, dim, lens = 2, 64, [3000, 900, 5000, 2000]
    cache = _kv.random_cache(lens, heads, dim, dtype, cuda, seed=5, weights=True)
    q = make_rows(9, heads * per * dim, dtype, cuda, 6)
    rows = _kv.rows(q, heads * per, dim)
    good = _kv.starts_of([2, 3, 2, 2], cuda)
    want = torch.empty_like(q)
    ops.attention_cached(rows, cache, good, want)
    wait(cuda)
    for bad in ([0, 9, 0, 9, 9], [0, 9, 1, 9, 2], [5, 0, 9, 3, 9]):
        ops.attention_cached(rows, cache, torch.tensor(bad, dtype=torch.int32, device=cuda), torch.empty_like(q), accumulate=True)
        with pytest.raises(native.H3Error, match="starts"):
            wait(cuda)
    out = torch.empty_like(q)
    ops.attention_cached(rows, cache, good, out)
    wait(cuda)
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_bad_pages_of_many_rows_and_of_an_append(dtype, cuda):
    heads, per, dim = 2, 2, 64
    cache = _kv.random_cache([700, 300], heads, dim, dtype, cuda, seed=7)
    q = make_rows(220, heads * per * dim, dtype, cuda, 8)
    starts = _kv.starts_of([120, 100], cuda)
    rows = _kv.rows(q, heads * per, dim)
    good = torch.empty_like(q)
    ops.attention_cached(rows, cache, starts, good)
    wait(cuda)
    page = int(cache.table[0, 3])
    for bad in (-1, cache.k.shape[0], 1 << 30, -(1 << 31)):
        cache.table[0, 3] = bad
        out = torch.empty_like(q)
        ops.attention_cached(rows, cache, starts, out)
        with pytest.raises(native.H3Error, match="page id"):
            wait(cuda)
        assert torch.equal(out[120:], good[120:])
    cache.table[0, 3] = page
    cache.table[1, 4:] = cache.k.shape[0]
    codes = cache.k.clone()
    cache.lens[1] = 330
    ops.kv_append(cache, _kv.rows(q, heads, dim), _kv.rows(q, heads, dim), torch.tensor([0, 0, 30], dtype=torch.int32, device=cuda))
    with pytest.raises(native.H3Error, match="page id"):
        wait(cuda)
    assert torch.equal(cache.k, codes)
