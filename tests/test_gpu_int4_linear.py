"""h3s_int4_linear and h3s_int4_pack on the GPU against the formula in 64 bits.

Tolerance: the products are exact (a code less 8 is, and x enters whole), so an output is off by its own rounding (half a
step of its type) and by the 32-bit sums: with A = sum |x| scale (|code - 8| + |zero - 8|), at most (K / 64 + 64) 2^-22 A: a warp
adds a few of every 64 products in a row, cutting off instead of rounding at most, then come the group's scale, the other
warps' sums and the bias."""
import pytest
import torch

from sycl_minimax_h3_b200 import native, ops

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(M, N, K, group, x_dt, s_dt, zero, bias, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    groups = -(-K // group) if group else 1
    codes = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    scale = (0.01 + 0.05 * torch.rand(groups, N, generator=g)).to(s_dt)
    z = (5 + 6 * torch.rand(groups, N, generator=g)).to(s_dt) if zero else None
    b = torch.randn(N, generator=g) if bias else None
    x = torch.randn(M, K, generator=g).to(x_dt)
    packed = (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous().to(device)
    lin = ops.Int4Linear.pack(packed, scale.to(device), group, None if z is None else z.to(device), None if b is None else b.to(device))
    return codes, scale, z, b, x, lin


def check(codes, scale, z, b, x, group, out):
    K = codes.shape[1]
    at = torch.arange(K) // (group or K)
    s = scale.double().t()[:, at]
    zero = torch.full_like(s, 8.0) if z is None else z.double().t()[:, at]
    w = s * (codes.double() - zero)
    xd = x.double()
    want = xd @ w.t() + (0 if b is None else b.double())
    A = xd.abs() @ (s * ((codes.double() - 8).abs() + (zero - 8).abs())).t() + (0 if b is None else b.double().abs())
    bound = (K / 64 + 64) * 2.0 ** -22 * A
    bound = bound + (want.abs() + bound) * (torch.finfo(out.dtype).eps / 2) + torch.finfo(out.dtype).tiny
    off = (out.double().cpu() - want).abs() - bound
    assert float(off.max()) <= 0, f"off by {float(off.max()):.3g} more than the roundings"


@pytest.mark.parametrize("x_dt", TYPES)
@pytest.mark.parametrize("group,zero", [(0, False), (32, True), (64, False), (128, True)])
@pytest.mark.parametrize("M,N,K", [(1, 16, 64), (1, 1, 2), (3, 33, 130), (8, 40, 512), (9, 100, 1000), (17, 64, 768), (70, 130, 448)])
def test_linear(x_dt, group, zero, M, N, K, cuda):
    s_dt = TYPES[(M + N) % 3]
    codes, scale, z, b, x, lin = make(M, N, K, group, x_dt, s_dt, zero, M % 2 == 1, cuda, seed=M + N + K)
    out = torch.empty(M, N, dtype=x_dt, device=cuda)
    lin.forward(x.to(cuda), out)
    ops.context(cuda).wait()
    check(codes, scale, z, b, x, group, out)


@pytest.mark.parametrize("x_dt", TYPES)
@pytest.mark.parametrize("out_dt", TYPES)
def test_output_types_and_unaligned_x(x_dt, out_dt, cuda):
    M, N, K = 5, 50, 264
    codes, scale, z, b, x, lin = make(M, N, K, 32, x_dt, torch.float32, True, True, cuda, seed=1)
    buf = torch.empty(M * K + 1, dtype=x_dt, device=cuda)
    buf[1:] = x.reshape(-1).to(cuda)
    room = torch.full((M * N + 5,), 7.0, dtype=out_dt, device=cuda)
    lin.forward(buf[1:].view(M, K), room[3:3 + M * N].view(M, N))
    ops.context(cuda).wait()
    check(codes, scale, z, b, x, 32, room[3:3 + M * N].view(M, N))
    assert bool((room[:3] == 7).all()) and bool((room[3 + M * N:] == 7).all())


@pytest.mark.parametrize("M", [1, 4, 16, 33])
def test_long_and_wide(M, cuda):
    codes, scale, z, b, x, lin = make(M, 2000, 4096, 128, torch.bfloat16, torch.bfloat16, False, True, cuda, seed=2)
    out = torch.empty(M, 2000, dtype=torch.float32, device=cuda)
    lin.forward(x.to(cuda), out)
    ops.context(cuda).wait()
    check(codes, scale, z, b, x, 128, out)


def test_float32_keeps_all_its_bits(cuda):
    """x of 24 bits against codes that pick one input each: the output is x times the scale, to the last bit."""
    K, N = 64, 64
    codes = torch.full((N, K), 8, dtype=torch.uint8)
    codes[torch.arange(N), torch.arange(K)] = 9
    scale = torch.ones(1, N)
    packed = (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous().to(cuda)
    lin = ops.Int4Linear.pack(packed, scale.to(cuda), 0)
    x = torch.randn(2, K, generator=torch.Generator().manual_seed(3))
    x[0, :4] = torch.tensor([1 + 2.0 ** -23, -3.0e38, 1e-30, 0.0])
    out = torch.empty(2, N, device=cuda)
    lin.forward(x.to(cuda), out)
    ops.context(cuda).wait()
    assert torch.equal(out.cpu(), x)


@pytest.mark.parametrize("x_dt", TYPES)
def test_nan_and_infinity_stay_in_their_row(x_dt, cuda):
    codes, scale, z, b, x, lin = make(4, 32, 96, 32, x_dt, torch.float32, False, False, cuda, seed=4)
    x[1, 7], x[2, 9] = float("nan"), float("inf")
    out = torch.empty(4, 32, dtype=x_dt, device=cuda)
    lin.forward(x.to(cuda), out)
    ops.context(cuda).wait()
    assert bool(out[1].isnan().all()) and not bool(out[2].isfinite().any())
    w = scale.double().t()[:, torch.arange(96) // 32] * (codes.double() - 8)
    assert torch.equal(out[2].cpu().isnan(), (w[:, 9] == 0) | (x[2].double() @ w.t()).isnan())
    keep = [0, 3]
    check(codes, scale, z, b, x[keep], 32, out[keep])


def test_pack_is_the_documented_layout(cuda):
    """Lane (g, t), word w, nibble j + 4 e: output g + 8 (j % 2), input 32 (w / 2) + 8 t + 4 (w % 2) + 2 (j / 2) + e."""
    N, K = 19, 70
    codes = torch.randint(0, 16, (N, K), generator=torch.Generator().manual_seed(5), dtype=torch.uint8)
    lin = ops.Int4Linear.pack((codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous().to(cuda), torch.ones(1, N, device=cuda), 0)
    ops.context(cuda).wait()
    tiles = lin.tiles.cpu()
    for nt in range(2):
        for kt in range(2):
            for lane in range(32):
                for w in range(4):
                    word = int(tiles[nt, kt, lane * 4 + w]) & 0xffffffff
                    for j in range(4):
                        for e in range(2):
                            n = nt * 16 + lane // 4 + 8 * (j % 2)
                            k = kt * 64 + 32 * (w // 2) + 8 * (lane % 4) + 4 * (w % 2) + 2 * (j // 2) + e
                            assert (word >> (4 * (j + 4 * e))) & 15 == (int(codes[n, k]) if n < N and k < K else 8)


def test_refusals(cuda):
    ctx = ops.context(cuda)
    L = native.lib()
    call = lambda **kw: L.h3s_int4_linear(ctx.handle, *{**dict(x=16, x_dt=0, M=1, K=64, t=16, N=16, s=16, z=0, s_dt=0, group=32, b=0, o=16, o_dt=0), **kw}.values())  # noqa: E731
    assert call(M=0) == 0 and call(N=0) == 0 and call(K=0) == 0
    for kw, why in (({"group": 16}, "groups"), ({"x_dt": 3}, "type"), ({"t": 8}, "16 bytes"), ({"s": 0}, "null")):
        assert call(**kw) == -1 and why in native.last_error()


@pytest.mark.parametrize("x_dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group,zero", [(0, True), (32, True), (64, True), (128, True), (32, False), (128, False)])
@pytest.mark.parametrize("M,N,K,shift", [(17, 130, 14336, 0), (40, 130, 1344, 0), (65, 257, 2112, 0), (129, 16, 62, 0), (64, 128, 1026, 0), (33, 140, 4096, 1)])
def test_many_rows(x_dt, group, zero, M, N, K, shift, cuda):
    """More stages than the rings have, parts that end inside a stage, rows past 32 and 64, x that cannot be copied by 16 bytes"""
    codes, scale, z, b, x, lin = make(M, N, K, group, x_dt, torch.float32, zero, True, cuda, seed=M + K)
    buf = torch.empty(M * K + shift, dtype=x_dt, device=cuda)
    buf[shift:] = x.reshape(-1).to(cuda)
    out = torch.full((M + 1, N), 7.0, dtype=torch.float32, device=cuda)
    lin.forward(buf[shift:].view(M, K), out[:M])
    ops.context(cuda).wait()
    check(codes, scale, z, b, x, group, out[:M])
    assert (out[M] == 7.0).all()


def test_nan_and_infinity_stay_in_their_row_of_many(cuda):
    codes, scale, z, b, x, lin = make(40, 150, 1024, 128, torch.bfloat16, torch.bfloat16, False, False, cuda, seed=5)
    x[1, 7], x[33, 900] = float("nan"), float("inf")
    out = torch.empty(40, 150, dtype=torch.float32, device=cuda)
    lin.forward(x.to(cuda), out)
    ops.context(cuda).wait()
    bad = ~torch.isfinite(out).all(1).cpu()
    assert bad.nonzero().flatten().tolist() == [1, 33]
    keep = [m for m in range(40) if m not in (1, 33)]
    check(codes, scale, z, b, x[keep], 128, out[keep])


@pytest.mark.parametrize("M,N,K", [(17, 1, 8), (64, 128, 56), (40, 20, 72), (200, 33, 200)])
def test_many_rows_of_few_inputs(M, N, K, cuda):
    """Fewer inputs than a box of x has"""
    codes, scale, z, b, x, lin = make(M, N, K, 32, torch.float16, torch.float16, True, True, cuda, seed=M + K)
    out = torch.empty(M, N, dtype=torch.float32, device=cuda)
    lin.forward(x.to(cuda), out)
    ops.context(cuda).wait()
    check(codes, scale, z, b, x, 32, out)


@pytest.mark.parametrize("M", [4, 12, 40])
def test_captured_calls_read_what_x_holds_at_the_replay(M, cuda):
    codes, scale, z, b, x, lin = make(M, 300, 1024, 64, torch.bfloat16, torch.float32, True, True, cuda, seed=7)
    held, out = torch.zeros(M, 1024, dtype=torch.bfloat16, device=cuda), torch.empty(M, 300, device=cuda)
    stream, graph = torch.cuda.Stream(cuda), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        lin.forward(held, out)
    for i in range(3):
        xi = x.roll(i, 1)
        held.copy_(xi)
        graph.replay()
        torch.cuda.synchronize()
        check(codes, scale, z, b, xi, 64, out)
    eager = torch.empty_like(out)
    lin.forward(held, eager)
    ops.context(cuda).wait()
    assert torch.equal(eager, out)


@pytest.mark.parametrize("x_dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("group", [0, 32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(40, 9600, 14336), (17, 9600, 1280), (64, 200, 14336)])
def test_zero_points_over_many_stages(x_dt, group, M, N, K, cuda):
    """Codes that are all 8, so that the output is the zero points' part alone: scale (8 - zero) times the sum of x over a
    group. More stages than the rings have, in CTAs that take all of a layer's inputs and in parts of them; every call gives
    the same bits."""
    g = torch.Generator().manual_seed(M + K + group)
    groups = -(-K // group) if group else 1
    packed = torch.full((N, K // 2), 0x88, dtype=torch.uint8, device=cuda)
    s = (0.01 + 0.05 * torch.rand(groups, N, generator=g)).to(cuda)
    z = (5 + 6 * torch.rand(groups, N, generator=g)).to(cuda)
    # the stages' rows are unlike: another size for every 128 inputs
    size = 2.0 ** torch.randint(-3, 4, (1, K // 128), generator=g).repeat_interleave(128, 1)
    x = (torch.randn(M, K, generator=g) * size).to(x_dt).to(cuda)
    lin = ops.Int4Linear.pack(packed, s, group, z)
    out = torch.empty(M, N, device=cuda)
    lin.forward(x, out)
    ops.context(cuda).wait()
    part = s.double() * (8 - z.double())
    sums = x.double().view(M, groups, K // groups)
    want = sums.sum(2) @ part
    bound = (K / 64 + 64) * 2.0 ** -22 * (sums.abs().sum(2) @ part.abs())
    bound = bound + want.abs() * 2.0 ** -23 + torch.finfo(torch.float32).tiny
    assert float(((out.double() - want).abs() - bound).max()) <= 0
    again = torch.empty_like(out)
    for _ in range(20):
        lin.forward(x, again)
        ops.context(cuda).wait()
        assert torch.equal(again, out)


def by_definition(codes, scale, z, b, x, group):
    """The layer in 64 bits, term by term: infinities, NaN and 0 times infinity as they come."""
    K = codes.shape[1]
    at = torch.arange(K) // (group or K)
    s = scale.double().t()[:, at]
    w = codes.double() - (8.0 if z is None else z.double().t()[:, at])
    y = torch.stack([(s * (w * row)).sum(1) for row in x.double()])
    return y if b is None else y + b.double()


def check_with_infinities(codes, scale, z, b, x, group, out):
    """NaN and infinities where the definition rounded to the output's type has them; the rest within ``check``'s bound."""
    want = by_definition(codes, scale, z, b, x, group)
    got = out.cpu()
    rounded = want.float().to(out.dtype)
    assert torch.equal(got.isnan(), rounded.isnan())
    assert torch.equal(got.isinf(), rounded.isinf()) and torch.equal(got[got.isinf()], rounded[rounded.isinf()])
    at = torch.arange(codes.shape[1]) // (group or codes.shape[1])
    s = scale.double().t()[:, at]
    zero = torch.full_like(s, 8.0) if z is None else z.double().t()[:, at]
    A = (x.double().abs() @ (s.abs() * ((codes.double() - 8).abs() + (zero - 8).abs())).t()) + (0 if b is None else b.double().abs())
    bound = (codes.shape[1] / 64 + 64) * 2.0 ** -22 * A
    bound = bound + (want.abs() + bound) * (torch.finfo(out.dtype).eps / 2) + torch.finfo(out.dtype).tiny
    fin = rounded.isfinite()
    assert not bool(((got.double() - want).abs() > bound)[fin].any())


ROWS_OF_EACH_KERNEL = [(4, torch.bfloat16), (4, torch.float16), (4, torch.float32), (12, torch.bfloat16), (12, torch.float32),
                       (40, torch.bfloat16), (40, torch.float16), (40, torch.float32), (70, torch.float16)]


@pytest.mark.parametrize("M,x_dt", ROWS_OF_EACH_KERNEL)
@pytest.mark.parametrize("group,zero", [(0, True), (32, True), (64, True), (128, True), (32, False)])
def test_infinities_meet_zero_points(M, x_dt, group, zero, cuda):
    """An infinite input: its output is the infinity of (code - zero)'s sign, NaN only where code = zero or where two of them
    meet with unlike signs; one row of NaN, one with an infinity of each sign."""
    K, N = 328, 70
    codes, scale, z, b, x, lin = make(M, N, K, group, x_dt, torch.float32, zero, True, cuda, seed=M + group)
    if zero:
        z[:, 5] = 8.0                                  # zero points that are codes: 0 times infinity
        z[:, 6] = 3.0
        lin = ops.Int4Linear(lin.tiles, lin.scale, N, K, group, z.to(cuda), lin.bias)
    x[0, 7] = float("inf")
    x[1, 40] = -float("inf")
    x[2, 3], x[2, 100] = float("inf"), -float("inf")
    x[M - 1, 327] = float("nan")
    out = torch.empty(M, N, dtype=x_dt, device=cuda)
    lin.forward(x.to(cuda), out)
    ops.context(cuda).wait()
    check_with_infinities(codes, scale, z, b, x, group, out)
    assert bool(out[0].isinf().any()) and bool(out[M - 1].isnan().all())


@pytest.mark.parametrize("M,x_dt", [m for m in ROWS_OF_EACH_KERNEL if m[1] != torch.float16])
@pytest.mark.parametrize("group,zero", [(0, True), (32, False), (64, True), (128, False)])
def test_sums_that_only_pass_the_largest_float_on_their_way(M, x_dt, group, zero, cuda):
    """Inputs near the largest of their type with scales that bring the terms back: the outputs are the definition's."""
    K, N = 328, 70
    codes, scale, z, b, x, lin = make(M, N, K, group, x_dt, torch.float32, zero, True, cuda, seed=M + group + 1)
    scale = scale * 2.0 ** -10
    lin = ops.Int4Linear(lin.tiles, scale.to(cuda), N, K, group, lin.zero, lin.bias)
    x[0] = (x[0].float().clamp(-3, 3) * 1e38).to(x_dt)
    x[M - 1, 5], x[M - 1, 6] = 3e38, -3e38
    out = torch.empty(M, N, device=cuda)
    lin.forward(x.to(cuda), out)
    ops.context(cuda).wait()
    assert bool(by_definition(codes, scale, z, b, x, group).float().isfinite().all())
    check_with_infinities(codes, scale, z, b, x, group, out)


@pytest.mark.parametrize("M", [4, 12, 40])
def test_scales_and_zero_points_that_are_not_finite_stay_in_their_output(M, cuda):
    K, N = 200, 40
    codes, scale, z, b, x, lin = make(M, N, K, 64, torch.bfloat16, torch.float32, True, True, cuda, seed=M + 2)
    scale[1, 3], scale[2, 5], z[0, 7], z[3, 9] = float("inf"), float("nan"), float("inf"), float("nan")
    codes[codes == 8] = 9
    packed = (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous().to(cuda)
    lin = ops.Int4Linear.pack(packed, scale.to(cuda), 64, z.to(cuda), b.to(cuda))
    out = torch.empty(M, N, device=cuda)
    lin.forward(x.to(cuda), out)
    ops.context(cuda).wait()
    want = by_definition(codes, scale, z, b, x, 64).float()
    assert torch.equal(out.cpu().isnan(), want.isnan()) and torch.equal(out.cpu().isinf(), want.isinf())
    keep = [n for n in range(N) if n not in (3, 5, 7, 9)]
    check(codes[keep], scale[:, keep], z[:, keep], b[keep], x, 64, out[:, keep])


@pytest.mark.parametrize("x_dt", TYPES)
@pytest.mark.parametrize("group,zero", [(0, False), (32, True), (64, True), (128, False), (32, False)])
@pytest.mark.parametrize("M,N,K", [(1, 9473, 200), (8, 9500, 1030), (3, 12288, 64)])
def test_few_rows_of_wide_layers(x_dt, group, zero, M, N, K, cuda):
    """Enough outputs for two strips to a CTA, an odd number of strips among them"""
    codes, scale, z, b, x, lin = make(M, N, K, group, x_dt, torch.bfloat16, zero, True, cuda, seed=N + K)
    out = torch.full((M + 1, N), 7.0, dtype=torch.float32, device=cuda)
    lin.forward(x.to(cuda), out[:M])
    ops.context(cuda).wait()
    check(codes, scale, z, b, x, group, out[:M])
    assert bool((out[M] == 7.0).all())
