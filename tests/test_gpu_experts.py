"""GPU: the layers of experts -- grouped Dense products, dropout from the counter-based generator, the 8-bit
integer product -- against plain float64 implementations on the CPU, and ExpertStack, which runs them together.

Tolerances, fixed before the first run.  u = 2^-24.  A sum of n float32 additions is off by at most
5 sqrt(n) u S (S = sum of the |products|) but for one element in 10^5 (the probabilistic bound, lambda = 5); a
matrix instruction's additions and, for float32, the six piece products make n <= 1.5 K + 16.  float32's split leaves out
products below 3 2^-26 S.  The result is then rounded to its type: finfo.eps / 2 of it.  float32 results are also held to the
norm bound sqrt(n) u, which a missing piece product (2^-17 and up) cannot meet."""
import numpy as np
import pytest
import torch

from weather_model_amd import synth

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rows(seed, shape, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def close(got, ref, S, n, what, norm=True):
    """got (device) against ref (float64) whose terms have absolute sum S over n additions each."""
    got_t, ref = got.detach().cpu(), torch.as_tensor(ref)
    assert got_t.shape == ref.shape, what
    h = half_step(got_t.dtype)
    acc = (5 * (1.5 * n + 16) ** 0.5 * U + 3 * 2.0 ** -26) * torch.as_tensor(S, dtype=torch.float64)
    tiny = torch.finfo(got_t.dtype).tiny
    bad = (got_t.double() - ref).abs() > (1 + h) * acc + h * ref.abs() + tiny
    assert not bool(bad.any()), (what, int(bad.sum()), float((got_t.double() - ref).abs().max()))
    if norm and got_t.dtype == torch.float32 and float(ref.norm()) > 0:
        assert float((got_t.double() - ref).norm() / ref.norm()) <= (1.5 * n + 16) ** 0.5 * U, what


def offsets_of(sizes, before=0):
    return torch.tensor(np.cumsum([before] + list(sizes)), dtype=torch.int64, device="cuda")


def grouped_ref(x, w, b, sizes, before, relu):
    """(y, S) in float64 on the CPU"""
    y = torch.zeros((x.shape[0], w.shape[1]), dtype=torch.float64)
    S = torch.zeros_like(y)
    at = before
    for g, n in enumerate(sizes):
        p = slice(at, at + n)
        y[p] = x[p].double() @ w[g].double().t()
        S[p] = x[p].double().abs() @ w[g].double().abs().t()
        if b is not None:
            y[p] += b[g].double()
            S[p] += b[g].double().abs()
        at += n
    return (y.clamp(min=0) if relu else y), S


SHAPES = [
    # sizes, N, K, rows before, rows behind
    ([1], 4, 4, 0, 0),
    ([1], 8000, 640, 0, 0),
    ([5, 0, 3, 130], 37, 19, 0, 0),
    ([0, 0, 0], 16, 16, 3, 2),                     # nobody has rows
    ([128, 256, 1], 128, 64, 0, 0),
    ([129, 127, 0, 383], 216, 432, 2, 5),          # singleRegression's map
    ([300] + [0] * 63 + [40], 65, 129, 0, 1),      # more than one wave of groups
    (list(range(80)), 33, 40, 1, 0),
    ([700, 900], 300, 520, 0, 0),
    ([17, 2], 1, 1, 0, 0),
    ([600, 0, 1100], 520, 136, 2, 1),              # tiles of 256 x 256 and what is left behind them; K no multiple of a stage
    ([513, 700], 771, 88, 0, 0),                   # the same with columns that are no multiple of 16 bytes
    ([900], 1032, 1000, 0, 9),
    ([40] * 21, 72, 96, 0, 0),                     # quarters of small tiles
    ([3] * 30, 260, 64, 0, 4),
    ([900, 1200], 2056, 136, 1, 0),                # tiles of 256 x 256 forward, halves of them
    ([1100, 1000], 136, 2056, 0, 2),               # and backward
    ([2048], 2048, 72, 0, 0),                      # quarters
    ([33, 40], 2064, 4104, 0, 0),                  # gradients of weights in tiles of 256 x 256
    ([70, 0, 131], 40, 3000, 2, 1),                # few tiles and a long contraction: in parts, forward
    ([70, 0, 131], 3001, 41, 2, 1),                # and backward
    ([3], 1100, 96, 0, 0),
    ([300] * 3, 24, 1096, 0, 0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_grouped_forward(case, dtype):
    from weather_model_amd import ops
    sizes, N, K, before, behind = SHAPES[case]
    M = before + sum(sizes) + behind
    x, w, b = rows(case, (M, K), dtype), rows(case + 50, (len(sizes), N, K), dtype, K ** -0.5), rows(case + 90, (len(sizes), N), dtype, 0.3)
    off = offsets_of(sizes, before)
    for bias, relu in ((None, False), (b, True)):
        y = ops.dense_grouped_forward(x.cuda(), w.cuda(), off, None if bias is None else bias.cuda(), relu=relu)
        ref, S = grouped_ref(x, w, bias, sizes, before, relu)
        close(y, ref, S, K, (case, relu))
        inside = torch.zeros(M, dtype=torch.bool)
        inside[before:before + sum(sizes)] = True
        assert not bool(y.cpu()[~inside].any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_grouped_backward(case, dtype):
    from weather_model_amd import ops
    sizes, N, K, before, behind = SHAPES[case]
    M, G = before + sum(sizes) + behind, len(sizes)
    x, w, gy = rows(case + 7, (M, K), dtype), rows(case + 57, (G, N, K), dtype, K ** -0.5), rows(case + 97, (M, N), dtype)
    off = offsets_of(sizes, before)
    gx, gw, gb = ops.dense_grouped_backward(x.cuda(), w.cuda(), off, gy.cuda(), mask_below=x.cuda())
    gx0, none, none2 = ops.dense_grouped_backward(x.cuda(), w.cuda(), off, gy.cuda(), need_gw=False)
    assert none is None and none2 is None
    rx, Sx = grouped_ref(gy, w.transpose(1, 2), None, sizes, before, False)
    close(gx0, rx, Sx, N, (case, "gx"))
    keep = (x > 0).double()
    close(gx, rx * keep, Sx * keep, N, (case, "gx masked"))
    at = before
    for g, n in enumerate(sizes):
        p = slice(at, at + n)
        a, c = gy[p].double(), x[p].double()
        close(gw[g], a.t() @ c, a.abs().t() @ c.abs(), n, (case, g, "gw"))
        close(gb[g], a.sum(0), a.abs().sum(0), n, (case, g, "gb"), norm=False)
        at += n


@pytest.mark.parametrize("N,K", [(24, 70), (216, 201)])
def test_grouped_weight_gradient_split_over_rows(N, K):
    """Few small weights and many rows: the rows are split over workgroups and joined in a fixed order."""
    from weather_model_amd import _lib, ops
    sizes = [9000, 0, 5001]
    assert _lib.lib().wm_dense_grouped_bwd_wb_workspace_bytes(3, sum(sizes), N, K, 0) > 0
    for dtype in TYPES:
        x, gy = rows(1, (sum(sizes), K), dtype), rows(2, (sum(sizes), N), dtype)
        w = torch.zeros((3, N, K), dtype=dtype, device="cuda")
        off = offsets_of(sizes)
        runs = [ops.dense_grouped_backward(x.cuda(), w, off, gy.cuda(), need_gx=False) for _ in range(2)]
        assert torch.equal(runs[0][1], runs[1][1]) and torch.equal(runs[0][2], runs[1][2])
        at = 0
        for g, n in enumerate(sizes):
            a, c = gy[at:at + n].double(), x[at:at + n].double()
            close(runs[0][1][g], a.t() @ c, a.abs().t() @ c.abs(), n, g)
            close(runs[0][2][g], a.sum(0), a.abs().sum(0), n, g, norm=False)
            at += n


def test_grouped_weight_gradient_of_one_expert_with_most_of_the_rows():
    """Many experts, one of which is cut in chunks; the others are not, or have no rows at all."""
    from weather_model_amd import ops
    sizes, N, K = [3] * 20 + [9001] + [0] * 10 + [40] * 9, 40, 72
    for dtype in TYPES:
        x, gy = rows(1, (sum(sizes), K), dtype), rows(2, (sum(sizes), N), dtype)
        w = torch.zeros((len(sizes), N, K), dtype=dtype, device="cuda")
        _, gw, gb = ops.dense_grouped_backward(x.cuda(), w, offsets_of(sizes), gy.cuda(), need_gx=False,
                                               out_w=torch.full_like(w, 7), out_b=torch.full((len(sizes), N), 7, dtype=dtype, device="cuda"))
        at = 0
        for g, n in enumerate(sizes):
            a, c = gy[at:at + n].double(), x[at:at + n].double()
            close(gw[g], a.t() @ c, a.abs().t() @ c.abs(), n, g)
            close(gb[g], a.sum(0), a.abs().sum(0), n, g, norm=False)
            at += n


def test_grouped_offsets_of_any_value_are_safe():
    from weather_model_amd import ops
    x, w = rows(1, (20, 8), torch.float32), rows(2, (4, 6, 8), torch.float32)
    for off, sizes, before in (([-5, 3, 2, 99, 7], [3, 0, 17, 0], 0), ([4, 4, 1, 6, 6], [0, 0, 2, 0], 4),
                               ([2 ** 40, 0, 0, 0, 0], [0, 0, 0, 0], 20)):
        y = ops.dense_grouped_forward(x.cuda(), w.cuda(), torch.tensor(off, device="cuda"))
        ref, S = grouped_ref(x, w, None, sizes, before, False)
        close(y, ref, S, 8, off)


def test_offsets_of_any_value_are_safe_in_every_path():
    """Few and many rows, chunks of rows, parts of a contraction, 8 bits: offsets outside 0 .. M and falling ones."""
    from weather_model_amd import ops
    for M, N, K in ((3, 20, 40), (60, 24, 72), (200, 40, 1100), (3000, 24, 40)):
        x, w, gy = rows(1, (M, K), torch.float32), rows(2, (4, N, K), torch.float32, K ** -0.5), rows(3, (M, N), torch.float32)
        raw = [-5, M - 2, 1, M + 99, 7]
        sizes = [M - 2, 0, 2, 0]
        off = torch.tensor(raw, device="cuda")
        y = ops.dense_grouped_forward(x.cuda(), w.cuda(), off)
        ref, S = grouped_ref(x, w, None, sizes, 0, False)
        close(y, ref, S, K, M)
        gx, gw, gb = ops.dense_grouped_backward(x.cuda(), w.cuda(), off, gy.cuda())
        rx, Sx = grouped_ref(gy, w.transpose(1, 2), None, sizes, 0, False)
        close(gx, rx, Sx, N, M)
        a, c = gy[:M - 2].double(), x[:M - 2].double()
        close(gw[0], a.t() @ c, a.abs().t() @ c.abs(), M, M)
        close(gb[0], a.sum(0), a.abs().sum(0), M, M, norm=False)
        assert not bool(gw[1].any()) and not bool(gw[3].any()) and not bool(gb[1].any())
        q, t = ops.quantize_rows(w.reshape(-1, K).cuda())
        y8 = ops.dense_i8(x.cuda(), q.view(4, N, K), t.view(4, N), offsets=off).cpu().double()
        xq, xs = codes_ref(x)
        for g, p in ((0, slice(0, M - 2)), (2, slice(M - 2, M))):
            e = (xq[p] @ q.view(4, N, K)[g].cpu().double().t()) * xs[p][:, None] * t.view(4, N)[g].cpu().double()
            assert bool(((y8[p] - e).abs() <= 5 * U * e.abs()).all()), (M, g)


def test_as_many_experts_as_there_may_be():
    from weather_model_amd import ops
    G, N, K = 4096, 12, 20
    sizes = torch.randint(0, 4, (G,), generator=torch.Generator().manual_seed(1)).tolist()
    sizes[77] = 600
    M = sum(sizes)
    x, w, gy = rows(1, (M, K), torch.bfloat16), rows(2, (G, N, K), torch.bfloat16, K ** -0.5), rows(3, (M, N), torch.bfloat16)
    off = offsets_of(sizes)
    y = ops.dense_grouped_forward(x.cuda(), w.cuda(), off)
    ref, S = grouped_ref(x, w, None, sizes, 0, False)
    close(y, ref, S, K, "y")
    gx, gw, gb = ops.dense_grouped_backward(x.cuda(), w.cuda(), off, gy.cuda())
    rx, Sx = grouped_ref(gy, w.transpose(1, 2), None, sizes, 0, False)
    close(gx, rx, Sx, N, "gx")
    at = np.cumsum([0] + sizes)
    for g in (0, 1, 63, 64, 77, 78, 2047, 4094, 4095):
        a, c = gy[at[g]:at[g + 1]].double(), x[at[g]:at[g + 1]].double()
        close(gw[g], a.t() @ c, a.abs().t() @ c.abs(), sizes[g], g)
        close(gb[g], a.sum(0), a.abs().sum(0), sizes[g], g, norm=False)


def test_strided_inputs_are_taken_as_their_values():
    from weather_model_amd import ops
    sizes, N, K = [40, 61], 24, 36
    off = offsets_of(sizes)
    x, w, gy = (rows(k, s, torch.bfloat16).cuda() for k, s in ((1, (101, K)), (2, (2, N, K)), (3, (101, N))))
    xs, ws, gs = x.t().contiguous().t(), w.transpose(0, 2).contiguous().transpose(0, 2), torch.cat([gy, gy], 1)[:, N:]
    assert not xs.is_contiguous() and not ws.is_contiguous() and not gs.is_contiguous()
    assert torch.equal(ops.dense_grouped_forward(x, w, off), ops.dense_grouped_forward(xs, ws, off))
    for a, b in zip(ops.dense_grouped_backward(x, w, off, gy, mask_below=x), ops.dense_grouped_backward(xs, ws, off, gs, mask_below=xs)):
        assert torch.equal(a, b)
    assert torch.equal(ops.dropout_forward(x, 0.4, 3, residual=x), ops.dropout_forward(xs, 0.4, 3, residual=xs))
    row = x[:1].expand(50, K)
    assert torch.equal(ops.quantize_rows(row)[0], ops.quantize_rows(row.contiguous())[0])
    bias = torch.ones((1, 1), dtype=torch.bfloat16, device="cuda").expand(2, N)
    assert torch.equal(ops.dense_grouped_forward(x, w, off, bias), ops.dense_grouped_forward(x, w, off, bias.contiguous()))


@pytest.mark.parametrize("more", [0, 230])
@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_infinities_and_nan_stay_in_their_rows(dtype, more):
    """An infinity or a NaN in a row, in a weight, in a row of no expert, next to zeros; float32 values that round up
    to infinity in bf16: the results are those of the arithmetic itself."""
    from weather_model_amd import ops
    inf, nan = float("inf"), float("nan")
    M, A = 70 + more, 30 + more
    x, w = rows(1, (M, 48), dtype), rows(2, (2, 40, 48), dtype, 48 ** -0.5)
    x[3, 5], x[4, 6], x[5, 7], x[M - 1, 0], x[8, :] = inf, -inf, nan, nan, 0
    w[1, 2, 5] = inf
    if dtype == torch.float32:
        x[9, 1], w[0, 7, 1] = 3.4e38, 0.5
        x[10, :], w[0, 8, :] = 0.0, 0.0           # a product next to the largest value
        x[10, 2] = w[0, 8, 2] = 1.84467429e19
    sizes = [A, 39]
    gy = rows(3, (M, 40), dtype)
    gy[6, 1], gy[M - 1, 2] = inf, nan
    y = ops.dense_grouped_forward(x.cuda(), w.cuda(), offsets_of(sizes))
    gx, gw, gb = ops.dense_grouped_backward(x.cuda(), w.cuda(), offsets_of(sizes), gy.cuda())
    xd, wd, gd = (t.double() for t in (x, w, gy))
    ry = torch.cat([xd[:A] @ wd[0].t(), xd[A:M - 1] @ wd[1].t(), torch.zeros(1, 40, dtype=torch.float64)])
    rx = torch.cat([gd[:A] @ wd[0], gd[A:M - 1] @ wd[1], torch.zeros(1, 48, dtype=torch.float64)])
    rw = torch.stack([gd[:A].t() @ xd[:A], gd[A:M - 1].t() @ xd[A:M - 1]])
    rb = torch.stack([gd[:A].sum(0), gd[A:M - 1].sum(0)])
    # sums of the absolute terms, which bound the finite results as everywhere (the module's tolerances)
    xa, wa, ga = (torch.where(t.isfinite(), t.abs(), 0.0) for t in (xd, wd, gd))
    zero = torch.zeros(1, 48, dtype=torch.float64)
    Sy = torch.cat([xa[:A] @ wa[0].t(), xa[A:M - 1] @ wa[1].t(), zero[:, :40]])
    Sx = torch.cat([ga[:A] @ wa[0], ga[A:M - 1] @ wa[1], zero])
    Sw = torch.stack([ga[:A].t() @ xa[:A], ga[A:M - 1].t() @ xa[A:M - 1]])
    Sb = torch.stack([ga[:A].sum(0), ga[A:M - 1].sum(0)])
    for name, got, ref, S, n in (("y", y, ry, Sy, 48), ("gx", gx, rx, Sx, 40), ("gw", gw, rw, Sw, A), ("gb", gb, rb, Sb, A)):
        got = got.cpu()
        ref = torch.where(ref.abs() > torch.finfo(dtype).max, ref.sign() * inf, ref)
        assert torch.equal(got.isnan(), ref.isnan()), name
        assert torch.equal(got.isposinf(), ref.isposinf()) and torch.equal(got.isneginf(), ref.isneginf()), name
        fine = ref.isfinite()
        close(got[fine], ref[fine], S[fine], n, name, norm=False)


@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** 60, 2.0 ** -120])
def test_grouped_float32_at_far_scales(scale):
    """The split keeps float32 accuracy from far below to far above 1 (2^-120: the third piece is subnormal in bf16,
    2^-133 is its last step: absolute error 2^-134 of each factor)."""
    from weather_model_amd import ops
    x, w = rows(1, (40, 64), torch.float32), rows(2, (1, 24, 64), torch.float32, 0.125)
    y = ops.dense_grouped_forward((x * scale).cuda(), w.cuda(), offsets_of([40]))
    ref, S = grouped_ref(x.double() * scale, w, None, [40], 0, False)
    d = (y.cpu().double() - ref).abs()
    assert bool((d <= (5 * 112 ** 0.5 * U + 3 * 2.0 ** -26) * S + 64 * 2.0 ** -133).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_takes_views_streams_and_unaligned_storage(dtype):
    """Strided views, storage that begins at an odd element, a side stream."""
    from weather_model_amd import ops
    sizes, N, K = [70, 60], 50, 33
    x, w, b = rows(1, (130, K), dtype), rows(2, (2, N, K), dtype, 0.2), rows(3, (2, N), dtype)
    ref, S = grouped_ref(x, w, b, sizes, 0, False)
    wide = torch.zeros((130, 2 * K), dtype=dtype)
    wide[:, ::2] = x
    flat = torch.zeros((x.numel() + 1,), dtype=dtype, device="cuda")
    flat[1:] = x.cuda().reshape(-1)
    wflat = torch.zeros((w.numel() + 1,), dtype=dtype, device="cuda")
    wflat[1:] = w.cuda().reshape(-1)
    wv = wflat[1:].view(w.shape)
    off = offsets_of(sizes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = ops.dense_grouped_forward(x.cuda(), w.cuda().transpose(1, 2).contiguous().transpose(1, 2), off, b.cuda())
    torch.cuda.current_stream().wait_stream(side)
    for y in (ys, ops.dense_grouped_forward(wide.cuda()[:, ::2], wv, off, b.cuda()),
              ops.dense_grouped_forward(flat[1:].view(130, K), wv, off, b.cuda())):
        close(y, ref, S, K, dtype)
    gy = rows(4, (130, N), dtype)
    gflat = torch.zeros((gy.numel() + 1,), dtype=dtype, device="cuda")
    gflat[1:] = gy.cuda().reshape(-1)
    got = ops.dense_grouped_backward(flat[1:].view(130, K), wv, off, gflat[1:].view(130, N))
    want = ops.dense_grouped_backward(x.cuda(), w.cuda(), off, gy.cuda())
    for a, c in zip(got, want):
        assert torch.equal(a, c)


def test_grouped_autograd_against_differences():
    """Gradients of a scalar of y against central differences of the float64 formula (step 1e-4: its own
    error is 1e-8 of the third derivative, zero for these products, plus 1e-12)."""
    from weather_model_amd import ops
    sizes, N, K = [4, 0, 9], 6, 5
    x, w, b, c = rows(1, (13, K), torch.float32), rows(2, (3, N, K), torch.float32), rows(3, (3, N), torch.float32), rows(4, (13, N), torch.float32)
    leaves = [t.clone().cuda().requires_grad_() for t in (x, w, b)]
    y = ops.dense_grouped(leaves[0], leaves[1], offsets_of(sizes), leaves[2], relu=True)
    (y * c.cuda()).sum().backward()

    def loss(xd, wd, bd):
        return float((grouped_ref(xd, wd, bd, sizes, 0, True)[0] * c.double()).sum())
    base = [t.double() for t in (x, w, b)]
    gen = torch.Generator().manual_seed(9)
    for k, leaf in enumerate(leaves):
        for _ in range(12):
            e = torch.zeros(base[k].numel(), dtype=torch.float64)
            at = int(torch.randint(base[k].numel(), (1,), generator=gen))
            e[at] = 1e-4
            d = (loss(*[t + e.view(t.shape) if j == k else t for j, t in enumerate(base)])
                 - loss(*[t - e.view(t.shape) if j == k else t for j, t in enumerate(base)])) / 2e-4
            assert abs(float(leaf.grad.reshape(-1)[at]) - d) <= 1e-5 * max(1.0, abs(d)), (k, at)


@pytest.mark.parametrize("dtype", TYPES)
def test_grouped_results_do_not_depend_on_where_the_tensors_lie(dtype):
    """The same rows in 16-byte rows (memory to LDS directly) and moved by one element (through registers): each within
    the bound of the other's sum; and run to run bit for bit."""
    from weather_model_amd import ops
    sizes, N, K = [130, 0, 300, 77], 144, 200
    M, G = sum(sizes), len(sizes)
    x, w, gy = rows(1, (M, K), dtype), rows(2, (G, N, K), dtype, K ** -0.5), rows(3, (M, N), dtype)

    def moved(t):
        flat = torch.zeros((t.numel() + 1,), dtype=dtype, device="cuda")
        flat[1:] = t.cuda().reshape(-1)
        return flat[1:].view(t.shape)
    off = offsets_of(sizes)
    outs = []
    for f in (lambda t: t.cuda(), moved, lambda t: t.cuda()):
        a = [f(t) for t in (x, w, gy)]
        outs.append([ops.dense_grouped_forward(a[0], a[1], off), *ops.dense_grouped_backward(a[0], a[1], off, a[2])])
    ref, S = grouped_ref(x, w, None, sizes, 0, False)
    close(outs[0][0], ref, S, K, "aligned")
    close(outs[1][0], ref, S, K, "moved")
    for a, b in zip(outs[0], outs[2]):
        assert torch.equal(a, b)


def test_grouped_offsets_and_storage_beyond_32_bits():
    """More than 2^31 elements of rows, and of weights: the last ones, and the first, against float64."""
    from weather_model_amd import ops
    M, K, N = 36000, 65536, 24
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty((M, K), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    w = torch.empty((2, N, K), dtype=torch.bfloat16, device="cuda").normal_(generator=gen) * K ** -0.5
    off = torch.tensor([0, 35990, M - 1], device="cuda")
    y = ops.dense_grouped_forward(x, w, off)
    some = [0, 17999, 35989, 35990, M - 2]
    for r in some:
        a, c = x[r].double().cpu(), w[int(r >= 35990)].double().cpu()
        close(y[r], c @ a, c.abs() @ a.abs(), K, r)
    assert not bool(y[M - 1].any())
    gy = torch.empty((M, N), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    _, gw, _ = ops.dense_grouped_backward(x, w, off, gy, need_gx=False, need_bias=False)
    for k in (0, K - 1):
        a, c = gy[35990:M - 1].double().cpu(), x[35990:M - 1, k].double().cpu()
        close(gw[1, :, k], a.t() @ c, a.abs().t() @ c.abs(), M, k)
    gx, _, _ = ops.dense_grouped_backward(x, w, off, gy, need_gw=False)
    a, c = gy[M - 2].double().cpu(), w[1].double().cpu()
    close(gx[M - 2], a @ c, a.abs() @ c.abs(), N, "gx")
    del x, y, gx, gw
    G, N, K = 3, 24000, 32000                       # 2.3e9 weights
    w = torch.empty((G, N, K), dtype=torch.bfloat16, device="cuda").normal_(generator=gen) * K ** -0.5
    for M in (5, 200):                              # few rows, tiles
        x = torch.empty((M, K), dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
        y = ops.dense_grouped_forward(x, w, torch.tensor([0, 1, 2, M], device="cuda"))
        a, c = x[M - 1].double().cpu(), w[2, -40:].double().cpu()
        close(y[M - 1, -40:], c @ a, c.abs() @ a.abs(), K, M)
    q = torch.randint(-127, 128, (G, N, K), device="cuda", generator=gen, dtype=torch.int8)
    t = torch.ones((G, N), device="cuda")
    for M in (3, 200):
        x = torch.empty((M, K), dtype=torch.float32, device="cuda").normal_(generator=gen)
        y = ops.dense_i8(x, q, t, offsets=torch.tensor([0, 1, 2, M], device="cuda"))
        xq, xs = codes_ref(x[M - 1:].cpu())
        ref = (xq @ q[2, -40:].double().cpu().t()) * xs[:, None]
        assert bool(((y[M - 1:, -40:].cpu().double() - ref).abs() <= 4 * U * ref.abs()).all()), M


def test_refusals():
    from weather_model_amd import ops
    x, w, off = rows(1, (6, 8), torch.float32).cuda(), rows(2, (2, 4, 8), torch.float32).cuda(), offsets_of([4, 2])
    bad = [
        (ValueError, "expects", lambda: ops.dense_grouped_forward(x, w[0], off)),
        (ValueError, "expects", lambda: ops.dense_grouped_forward(x[:, :7], w, off)),
        (TypeError, "like the rows", lambda: ops.dense_grouped_forward(x, w.half(), off)),
        (TypeError, "float32, bfloat16 or float16", lambda: ops.dense_grouped_forward(x.double(), w, off)),
        (TypeError, "int64", lambda: ops.dense_grouped_forward(x, w, off.int())),
        (ValueError, "offsets", lambda: ops.dense_grouped_forward(x, w, off[:2])),
        (RuntimeError, "no CPU fallback", lambda: ops.dense_grouped_forward(x, w, off.cpu())),
        (ValueError, "bias", lambda: ops.dense_grouped_forward(x, w, off, torch.zeros(4, device="cuda"))),
        (ValueError, "contiguous", lambda: ops.dense_grouped_forward(x, w, off, out=torch.zeros(6, 8, device="cuda")[:, :4])),
        (ValueError, "shares memory", lambda: ops.dense_grouped_forward(x, rows(2, (2, 8, 8), torch.float32).cuda(), off, out=x)),
        (ValueError, "grad_output", lambda: ops.dense_grouped_backward(x, w, off, x)),
        (ValueError, "mask", lambda: ops.dense_grouped_backward(x, w, off, x[:, :4], mask_below=x[:, :4])),
        (ValueError, "residual", lambda: ops.dropout_forward(x, 0.1, 1, residual=x[:3])),
        (ValueError, "shares memory", lambda: ops.dropout_forward(x[:3], 0.1, 1, out=x.view(-1)[8:32].view(3, 8))),
        (ValueError, "expects", lambda: ops.quantize_rows(x[0])),
        (ValueError, "expects", lambda: ops.quantize_rows(x[:, :0])),
        (TypeError, "int8", lambda: ops.dense_i8(x, w[0], torch.ones(4, device="cuda"))),
        (ValueError, "scale", lambda: ops.dense_i8(x, w[0].to(torch.int8), torch.ones(3, device="cuda"))),
        (ValueError, "expects", lambda: ops.dense_i8(x, w.to(torch.int8), torch.ones(2, 4, device="cuda"))),
        (TypeError, "float32", lambda: ops.dense_i8(x, w[0].to(torch.int8), torch.ones(4, device="cuda"), torch.ones(4, device="cuda").half())),
    ]
    for k, (error, text, call) in enumerate(bad):
        with pytest.raises(error, match=text):
            call()
            raise AssertionError(f"case {k} was taken")
    from weather_model_amd._lib import WmError
    with pytest.raises(WmError, match="beyond"):
        ops.dense_grouped_forward(x, torch.zeros((4097, 4, 8), device="cuda"), torch.zeros(4098, dtype=torch.int64, device="cuda"))


def test_nothing_to_do():
    """No rows at all: empty results, gradients of zeros."""
    from weather_model_amd import ops
    x, w, off = torch.zeros((0, 8), device="cuda"), torch.ones((2, 4, 8), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    assert ops.dense_grouped_forward(x, w, off).shape == (0, 4)
    gx, gw, gb = ops.dense_grouped_backward(x, w, off, torch.zeros((0, 4), device="cuda"))
    assert gx.shape == (0, 8) and not bool(gw.any()) and not bool(gb.any())
    assert ops.dropout_forward(x, 0.5, 1).shape == (0, 8)
    assert ops.quantize_rows(x)[0].shape == (0, 8)
    assert ops.dense_i8(x, torch.ones((4, 8), dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")).shape == (0, 4)
    # rows, but none owned
    y = ops.dense_grouped_forward(torch.ones((70, 8), device="cuda"), w, off)
    assert not bool(y.any())


def test_operators_in_two_streams_and_in_graphs():
    """Two calls at once on two streams, then each captured into a graph of its own and replayed in turn with eager work in
    between: every result equals the eager one."""
    from weather_model_amd import ops
    sizes, N, K = [300, 0, 261, 40], 136, 264
    off = offsets_of(sizes)
    sets = []
    for k in range(2):
        x, w = rows(5 + k, (sum(sizes), K), torch.bfloat16).cuda(), rows(7 + k, (len(sizes), N, K), torch.bfloat16, 0.1).cuda()
        q, t = ops.quantize_rows(w.reshape(-1, K))
        sets.append((x, w, rows(9 + k, (sum(sizes), N), torch.bfloat16).cuda(), q.view(w.shape), t.view(len(sizes), N)))

    def work(k):
        x, w, gy, q, t = sets[k]
        return [ops.dense_grouped_forward(x, w, off), *ops.dense_grouped_backward(x, w, off, gy), ops.dropout_forward(x, 0.3, k),
                ops.dense_i8(x, q, t, offsets=off), ops.dense_grouped_forward(x[:20], w, off)]
    want = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for k, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(work(k))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))
    graphs, outs = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(k))
        graphs.append(g)
    for turn in range(4):
        for k in (0, 1) if turn % 2 else (1, 0):
            for o in outs[k]:
                o.fill_(float("nan"))
            graphs[k].replay()
        work(turn % 2)
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(u, v) for u, v in zip(a, b)), turn


def test_autograd_of_second_order_and_in_a_capture_is_refused():
    """Gradients of gradients, and autograd's backward pass while a stream is captured (here with an eager graph of the same
    leaves alive): refused, and everything goes on."""
    from weather_model_amd import ops
    x, w = rows(1, (70, 8), torch.float32).cuda().requires_grad_(), rows(2, (2, 4, 8), torch.float32).cuda().requires_grad_()
    off = offsets_of([40, 30])
    alive = ops.dense_grouped(x, w, off), ops.dropout(x, 0.5, 1)
    for y in (ops.dense_grouped(x, w, off), ops.dropout(x, 0.5, 1)):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    one = torch.ones((70, 4), device="cuda"), torch.ones((70, 8), device="cuda")
    for k, make in enumerate((lambda: ops.dense_grouped(x, w, off), lambda: ops.dropout(x, 0.5, 1))):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = make()
            with pytest.raises(RuntimeError, match="cannot be captured"):
                y.backward(one[k])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, alive[k])
    alive[0].sum().backward()
    close(w.grad[0, 1], x[:40].detach().cpu().double().sum(0), x[:40].detach().cpu().double().abs().sum(0), 40, "gw")


# ------------------------------------------------------------------ dropout

def kept(n, p, seed, offset):
    """The documented draw in numpy: 16 bits of the hash of (seed, e / 4) above 16 of the hash of that."""
    e = np.arange(n, dtype=np.uint64) + np.uint64(offset)
    z = synth.hash64(seed, e >> np.uint64(2))
    at = (e & np.uint64(3)) * np.uint64(16)
    u = ((z >> at) & np.uint64(0xFFFF)) << np.uint64(16) | ((synth.hash64(seed, z) >> at) & np.uint64(0xFFFF))
    return torch.from_numpy(u >= np.uint64(round(p * 2 ** 32)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,p,offset", [(1, 0.5, 0), (7, 0.3, 0), (4099, 0.1, 0), (4099, 0.1, 1), (100003, 0.9, 2), (65536, 0.5, 3),
                                        (262145, 2.0 ** -16, 8), (262144, 1e-9, 5), (50000, 1.0, 0), (50001, 0.0, 0),
                                        (30000, 0.25, 2 ** 33 + 5), (30000, 0.25, 2 ** 62 + 6)])
def test_dropout_matches_the_documented_draw(n, p, offset, dtype):
    from weather_model_amd import ops
    x, r = rows(n, (n,), dtype), rows(n + 1, (n,), dtype)
    keep = kept(n, p, 77, offset)
    scale = 0.0 if p == 1.0 else 1.0 / (1.0 - round(p * 2 ** 32) / 2 ** 32)
    ref = torch.where(keep, x.double() * scale, 0.0)
    for res in (None, r):
        y = ops.dropout_forward(x.cuda(), p, 77, offset=offset, residual=None if res is None else res.cuda()).cpu()
        want = ref if res is None else ref + res.double()
        # the scale and the product are rounded in float32 (2 u), the sum (u), the result to its type
        tol = 4 * U * (ref.abs() + (0 if res is None else res.double().abs())) + half_step(dtype) * want.abs() + torch.finfo(dtype).tiny
        assert bool(((y.double() - want).abs() <= tol).all())
        if res is None:
            assert torch.equal(y == 0, (~keep) | (x == 0)) or dtype == torch.float16
    dev = ops.dropout_forward(x.cuda(), p, 77, offset=torch.tensor([offset], device="cuda")).cpu()
    assert torch.equal(dev, ops.dropout_forward(x.cuda(), p, 77, offset=offset).cpu())
    g = ops.dropout_backward(r.cuda(), p, 77, offset=offset).cpu()
    assert torch.equal(g == 0, (~keep) | (r == 0)) or dtype == torch.float16


def test_dropout_drops_infinities_works_in_place_and_in_pieces():
    from weather_model_amd import ops
    n, p = 10007, 0.4
    x = torch.full((n,), float("nan"), device="cuda")
    keep = kept(n, p, 5, 0)
    y = ops.dropout_forward(x, p, 5).cpu()
    assert torch.equal(y.isnan(), keep) and not bool(y[~keep].any())
    z = rows(1, (n,), torch.bfloat16).cuda()
    whole = ops.dropout_forward(z, p, 5, offset=11)
    parts = torch.cat([ops.dropout_forward(z[a:b], p, 5, offset=11 + a) for a, b in ((0, 1), (1, 4098), (4098, n))])
    assert torch.equal(whole, parts)
    ops.dropout_forward(z, p, 5, offset=11, out=z)
    assert torch.equal(z, whole)
    share = float(kept(1 << 20, 0.1, 3, 0).double().mean())
    assert abs(share - 0.9) < 5 * (0.09 / 2 ** 20) ** 0.5


def test_dropout_of_more_than_2_32_elements():
    from weather_model_amd import ops
    n, p = 2 ** 32 + 1027, 0.2
    x = torch.ones((n,), dtype=torch.bfloat16, device="cuda")
    ops.dropout_forward(x, p, 6, offset=3, out=x)
    for at in (0, 2 ** 31 - 500, 2 ** 32 - 500):
        m = min(1500, n - at)
        assert torch.equal(x[at:at + m].cpu() != 0, kept(m, p, 6, 3 + at)), at


def test_dropout_autograd_and_graph_replays_with_a_device_offset():
    from weather_model_amd import ops
    x, r = rows(1, (64, 130), torch.float32).cuda().requires_grad_(), rows(2, (64, 130), torch.float32).cuda().requires_grad_()
    gy = rows(3, (64, 130), torch.float32).cuda()
    ops.dropout(x, 0.3, 9, 40, residual=r).backward(gy)
    assert torch.equal(r.grad, gy)
    assert torch.equal(x.grad, ops.dropout_backward(gy, 0.3, 9, 40))
    counter = torch.zeros((1,), dtype=torch.int64, device="cuda")
    src, dst = rows(4, (5001,), torch.float32).cuda(), torch.empty((5001,), device="cuda")
    ops.dropout_forward(src, 0.5, 2, offset=counter, out=dst)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.dropout_forward(src, 0.5, 2, offset=counter, out=dst)
        counter.add_(5001)
    for k in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dst, ops.dropout_forward(src, 0.5, 2, offset=5001 * k)), k
    lost = ops.dropout(x, 0.3, 9, counter)
    counter.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lost.sum().backward()


# ------------------------------------------------------------------ 8 bits

def codes_ref(x):
    """(codes float64, scale float64) by the definition: float32 scale, float32 quotient rounded to even"""
    top = x.double().abs().amax(1)
    scale = (top / 127).float().double()
    q = (x.double() / torch.where(scale > 0, scale, 1.0)[:, None]).float().double().round().clamp(-127, 127)
    return q * (scale > 0)[:, None], scale


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 16), (2, 640), (33, 1283), (4, 8192), (1, 20011), (70, 63), (1100, 500),
                                 (1100, 999), (4200, 1501), (300, 1501), (1100, 2500), (300, 2500), (1100, 5000), (1030, 8200)])
def test_quantize_rows(M, K, dtype):
    from weather_model_amd import ops
    x = rows(M + K, (M, K), dtype) * torch.logspace(-3, 2, M)[:, None].to(dtype)
    if M > 2:
        x[1] = 0
        x[2, K // 2:] = -x[2].abs().max()
    q, s = ops.quantize_rows(x.cuda())
    rq, rs = codes_ref(x)
    assert torch.equal(s.cpu().double(), rs)
    assert torch.equal(q.cpu().double(), rq)


def test_quantize_ties_extremes_and_bad_rows():
    from weather_model_amd import ops
    x = torch.zeros((6, 130))
    x[0, 0], x[0, 1:7] = 127.0, torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, 126.5])          # ties go to even
    x[1, 0], x[1, 1] = 1e-45, 3e-45                                                       # the scale underflows to zero
    x[2, 5], x[2, 6] = 2.6e-43, -1.4e-45                                                  # a subnormal scale
    x[3, 9], x[4, 129], x[5, 3] = float("inf"), float("nan"), 3e38
    q, s = ops.quantize_rows(x.cuda())
    q, s = q.cpu(), s.cpu()
    assert q[0, :7].tolist() == [127, 0, 2, 2, 0, -2, 126]
    rq, rs = codes_ref(x[[0, 1, 2, 5]])
    assert torch.equal(q[[0, 1, 2, 5]].double(), rq) and torch.equal(s[[0, 1, 2, 5]].double(), rs)
    assert bool(s[3:5].isnan().all()) and not bool(q[3:5].any())
    w, t = ops.quantize_rows(rows(3, (40, 130), torch.float32).cuda())
    y = ops.dense_i8(x.cuda(), w, t).cpu()
    assert bool(y[3:5].isnan().all()) and not bool(y[:3].isnan().any()) and not bool(y[5].isnan().any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 8000, 640), (3, 37, 19), (16, 64, 128), (17, 130, 257), (128, 128, 64), (200, 301, 515),
                                   (130, 260, 2049), (48, 129, 33), (300, 50, 127), (600, 520, 272), (2048, 2048, 64), (2100, 2056, 272), (1, 40, 8192),
                                   (1, 33, 8200), (1, 17, 4099), (20, 300, 640), (2, 40, 8192), (4, 50, 8100), (5, 60, 2048), (16, 30, 2041), (9, 300, 1001),
                                   (3, 5000, 999), (2, 20, 9000), (16, 4100, 2048)])
def test_dense_i8(M, N, K, dtype):
    from weather_model_amd import ops
    x, b = rows(M, (M, K), dtype), rows(N, (N,), torch.float32)
    q, t = ops.quantize_rows(rows(K, (N, K), torch.float32, K ** -0.5).cuda())
    xq, xs = codes_ref(x)
    exact = (xq @ q.cpu().double().t()) * xs[:, None] * t.cpu().double()
    for bias, relu in ((None, False), (b, True)):
        y = ops.dense_i8(x.cuda(), q, t, None if bias is None else bias.cuda(), relu=relu).cpu()
        ref = exact if bias is None else exact + bias.double()
        ref = ref.clamp(min=0) if relu else ref
        # the integer, two scalings and the sum are rounded once each in float32
        tol = 4 * U * (exact.abs() + (0 if bias is None else bias.double().abs())) + half_step(dtype) * ref.abs() + torch.finfo(dtype).tiny
        assert bool(((y.double() - ref).abs() <= tol * (1 + 2.0 ** -8)).all())


@pytest.mark.parametrize("K", [70, 2100, 8191])
@pytest.mark.parametrize("sizes", [[1, 0, 3], [0, 2, 0, 0, 1], [9, 0, 4, 0, 2], [40, 0, 0, 3, 20]])
def test_dense_i8_few_rows_of_experts(sizes, K):
    from weather_model_amd import ops
    M, N, G = sum(sizes) + 1, 37, len(sizes)
    x, b = rows(K, (M, K), torch.bfloat16), rows(2, (G, N), torch.float32)
    q = torch.randint(-127, 128, (G, N, K), generator=torch.Generator().manual_seed(3)).to(torch.int8).cuda()
    t = rows(4, (G, N), torch.float32).abs().cuda()
    y = ops.dense_i8(x.cuda(), q, t, b.cuda(), offsets=offsets_of(sizes)).cpu().double()
    xq, xs = codes_ref(x)
    at = 0
    for g, n in enumerate(sizes):
        p = slice(at, at + n)
        e = (xq[p] @ q[g].cpu().double().t()) * xs[p][:, None] * t[g].cpu().double()
        ref = e + b[g].double()
        assert bool(((y[p] - ref).abs() <= 4 * U * (e.abs() + b[g].double().abs()) + 2.0 ** -8 * ref.abs()).all()), g
        at += n
    assert not bool(y[at:].any())


def test_dense_i8_grouped_extreme_codes_and_unaligned_weights():
    from weather_model_amd import ops
    sizes, N, K = [0, 50, 1, 0, 140], 45, 203
    M = sum(sizes) + 4
    x, b = rows(1, (M, K), torch.bfloat16), rows(2, (5, N), torch.float32)
    flat = torch.randint(-128, 128, (5 * N * K + 1,), generator=torch.Generator().manual_seed(3)).to(torch.int8).cuda()
    q = flat[1:].view(5, N, K)                                # storage begins at an odd byte; -128 among the codes
    t = rows(4, (5, N), torch.float32).abs().cuda()
    y = ops.dense_i8(x.cuda(), q, t, b.cuda(), offsets=offsets_of(sizes)).cpu().double()
    xq, xs = codes_ref(x)
    at = 0
    for g, n in enumerate(sizes):
        p = slice(at, at + n)
        e = (xq[p] @ q[g].cpu().double().t()) * xs[p][:, None] * t[g].cpu().double()
        ref = e + b[g].double()
        assert bool(((y[p] - ref).abs() <= 4 * U * (e.abs() + b[g].double().abs()) + 2.0 ** -8 * ref.abs()).all()), g
        at += n
    assert not bool(y[at:].any())
    # every product at its largest, over the longest sum that is allowed
    K = 1 << 17
    big = torch.full((2, K), -128, dtype=torch.int8, device="cuda")
    y = ops.dense_i8(torch.ones((1, K), device="cuda"), big, torch.ones((2,), device="cuda"))
    assert torch.equal(y.cpu(), torch.full((1, 2), float(np.float32(-127.0 * 128 * K) * (np.float32(1) / np.float32(127)))))


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("dtype", TYPES)
def test_expert_stack_trains_and_serves(dtype):
    """Three layers of four experts with dropout: activations and all gradients against the same chain in float64 on
    the layer's own inputs, a graph of the step replayed, then served in 8 bits within the codes' resolution."""
    from weather_model_amd.experts import ExpertStack
    sizes, widths, p = [40, 0, 133, 20], [20, 48, 33, 10], 0.25
    M, G = sum(sizes) + 3, len(sizes)
    x = rows(1, (M, widths[0]), dtype)
    ws = [rows(10 + l, (G, n, k), dtype, k ** -0.5) for l, (k, n) in enumerate(zip(widths, widths[1:]))]
    bs = [rows(20 + l, (G, n), dtype, 0.1) for l, n in enumerate(widths[1:])]
    gout = rows(30, (M, widths[-1]), dtype)
    off = offsets_of(sizes)
    st = ExpertStack([w.cuda() for w in ws], [b.cuda() for b in bs], p=p, seed=4)
    st.forward(x.cuda(), off, train=True)
    flat = st.backward(gout.cuda()).clone()
    h = [t.cpu() for t in st.h]
    scale = 1.0 / (1.0 - p)
    masks = []
    for l in range(3):
        ref, S = grouped_ref(h[l], ws[l], bs[l], sizes, 0, l < 2)
        if l < 2:
            keep = kept(ref.numel(), p, 4, (l << 48) + M * max(widths[1:-1])).view(ref.shape)
            ref, S = torch.where(keep, ref * scale, 0.0), S * scale
            masks.append((h[l + 1] > 0).double() * scale)
            # two roundings to the type: the product's and dropout's
            d = (h[l + 1].double() - ref).abs()
            assert bool((d <= 2.1 * half_step(dtype) * ref.abs() + 6 * 100 ** 0.5 * U * S + torch.finfo(dtype).tiny).all()), l
            assert not bool(h[l + 1][~keep].any())
        else:
            close(st.h[3], ref, S, widths[l], l)
    # the chain of gradients rounds to the type at every layer: at most (2 per layer) half steps of |.| propagated
    g, err = gout.double(), torch.zeros_like(gout, dtype=torch.float64)
    for l in range(2, -1, -1):
        at = 0
        ng, nerr = torch.zeros_like(h[l], dtype=torch.float64), torch.zeros_like(h[l], dtype=torch.float64)
        for e, n in enumerate(sizes):
            q = slice(at, at + n)
            a, c, w = g[q], h[l][q].double(), ws[l][e].double()
            u = 6 * (1.5 * max(n, widths[l + 1]) + 16) ** 0.5 * U
            tol = err[q].t() @ c.abs() + (a.abs() + err[q]).t() @ c.abs() * u + half_step(dtype) * (a.t() @ c).abs()
            assert bool(((st.gw[l][e].cpu().double() - a.t() @ c).abs() <= 1.01 * tol + torch.finfo(dtype).tiny).all()), (l, e)
            tol = err[q].sum(0) + a.abs().sum(0) * u + half_step(dtype) * a.sum(0).abs()
            assert bool(((st.gb[l][e].cpu().double() - a.sum(0)).abs() <= 1.01 * tol + torch.finfo(dtype).tiny).all()), (l, e)
            if l:
                ng[q] = a @ w * masks[l - 1][q]
                nerr[q] = (err[q] @ w.abs() + u * (a.abs() @ w.abs())) * masks[l - 1][q] + 2.1 * half_step(dtype) * ng[q].abs()
            at += n
        g, err = ng, 1.01 * nerr
    # the same step captured and replayed: every replay draws what the eager step in its place draws
    begin = torch.arange(2, device="cuda") << 48
    sx, sg = x.cuda(), gout.cuda()
    st.drawn.copy_(begin)
    eager = [st.step_grads(sx, off, sg).clone() for _ in range(3)]
    assert torch.equal(eager[0], flat) and not torch.equal(eager[1], flat)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        st.step_grads(sx, off, sg)
    st.drawn.copy_(begin)
    for want in eager:
        st.flat_grads.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(st.flat_grads, want)
    st.drawn.copy_(begin)
    # served: every code is within half a step of its value
    y8 = st.quantize().predict(x.cuda(), off).cpu().double()
    a, err = x.double(), torch.zeros_like(x, dtype=torch.float64)
    for l in range(3):
        z, S = grouped_ref(a, ws[l], bs[l], sizes, 0, False)
        z8, e8 = torch.zeros_like(z), torch.zeros_like(z)
        at = 0
        for e, n in enumerate(sizes):
            q = slice(at, at + n)
            dx = err[q] + (a[q].abs() + err[q]).amax(1, keepdim=True) / 254 * 1.001
            dw = ws[l][e].double().abs().amax(1, keepdim=True) / 254 * 1.001
            w = ws[l][e].double().abs()
            e8[q] = dx @ (w + dw).t() + a[q].abs() @ dw.expand_as(w).t()
            at += n
        z = z.clamp(min=0) if l < 2 else z
        e8 = e8 + half_step(dtype) * (z.abs() + e8) + 8 * U * (S + e8) + torch.finfo(dtype).tiny
        a, err = z, e8
    assert bool(((y8 - a).abs() <= 1.01 * err).all())
    assert float((y8 - a).norm() / a.norm()) < 0.05


def apart(spans):
    """Whether no two of the (begin, length) share an element."""
    spans = sorted(spans)
    return all(a + n <= b for (a, n), (b, _) in zip(spans, spans[1:]))


def test_expert_stack_draws_no_element_twice():
    """Steps of unlike numbers of rows -- the last batch of an epoch is shorter --, eager ones and replays of a graph in
    turn: each draws from where its `drawn` says, and no two from the same elements."""
    from weather_model_amd.experts import ExpertStack
    widths, p, seed = [20, 48, 33, 10], 0.25, 6
    st = ExpertStack([rows(10 + l, (2, n, k), torch.float32, k ** -0.5).cuda() for l, (k, n) in enumerate(zip(widths, widths[1:]))],
                     [rows(20 + l, (2, n), torch.float32, 0.1).cuda() for l, n in enumerate(widths[1:])], p=p, seed=seed)
    spans = [[], []]

    def seen(M):
        for l, at in enumerate(st.drawn.tolist()):
            n = M * widths[l + 1]
            keep = kept(n, p, seed, at).view(M, widths[l + 1])
            assert not bool(st.h[l + 1].cpu()[~keep].any()), (l, M)
            spans[l].append((at, n))
            assert apart(spans[l]), (l, M, spans[l])
    def step(M):
        off = torch.tensor([0, M // 3, M], device="cuda")
        return st.step_grads(rows(M, (M, widths[0]), torch.float32).cuda(), off, rows(M + 1, (M, widths[-1]), torch.float32).cuda())
    for M in (100, 7, 3, 64, 1, 1, 90):
        step(M)
        seen(M)
    M = 40
    sx, sg, off = rows(1, (M, widths[0]), torch.float32).cuda(), rows(2, (M, widths[-1]), torch.float32).cuda(), offsets_of([13, 27])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        st.step_grads(sx, off, sg)
    captured = st.h
    for other in (200, 5, 0, 1):
        graph.replay()
        torch.cuda.synchronize()
        st.h = captured
        seen(M)
        if other:
            step(other)
            seen(other)


@pytest.mark.parametrize("dtype", TYPES)
def test_expert_stack_serves_the_weights_and_biases_it_quantised(dtype):
    """Training that goes on in place does not reach what `predict` answers with."""
    from weather_model_amd.experts import ExpertStack
    widths = [24, 40, 9]
    ws = [rows(10 + l, (2, n, k), dtype, k ** -0.5).cuda() for l, (k, n) in enumerate(zip(widths, widths[1:]))]
    bs = [rows(20 + l, (2, n), dtype).cuda() for l, n in enumerate(widths[1:])]
    x, off = rows(1, (50, widths[0]), dtype).cuda(), offsets_of([20, 30])
    st = ExpertStack(ws, bs).quantize()
    before = st.predict(x, off).clone()
    for t in ws + bs:
        t.add_(1.0)
    assert torch.equal(st.predict(x, off), before)
    assert not torch.equal(st.quantize().predict(x, off), before)


def test_sizes_beyond_32_bits_are_refused():
    """A count that the C interface could only take modulo 2^32; the tensors are views of one element."""
    from weather_model_amd import ops
    n = 2 ** 32 + 4

    def view(*shape, dtype=torch.bfloat16):
        return torch.zeros((1,) * len(shape), dtype=dtype, device="cuda").expand(shape)
    one, off = view(1, 1, 1), offsets_of([4])
    calls = [lambda: ops.dense_grouped_forward(view(n, 1), one, off), lambda: ops.dense_grouped_forward(view(4, n), view(1, 1, n), off),
             lambda: ops.dense_grouped_forward(view(4, 1), view(1, n, 1), off),
             lambda: ops.dense_grouped_backward(view(n, 1), one, off, view(n, 1)), lambda: ops.quantize_rows(view(n, 1)),
             lambda: ops.dense_i8(view(n, 1), view(1, 1, dtype=torch.int8), view(1, dtype=torch.float32)),
             lambda: ops.dense_i8(view(4, 1), view(n, 1, dtype=torch.int8), view(n, dtype=torch.float32))]
    for k, call in enumerate(calls):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        with pytest.raises(ValueError, match="beyond 32 bits"):
            call()
            raise AssertionError(f"call {k} was taken")
        assert torch.cuda.max_memory_allocated() < before + (1 << 20), k          # nothing was copied first


# (sizes, N, K): few rows, small tiles, a contraction in parts forward and backward, chunks of rows, whole tiles
FAR = [([16], 24, 64), ([40], 24, 64), ([70, 0, 131], 40, 1100), ([70, 131], 1101, 41), ([2000, 0, 1501], 24, 40), ([300, 277], 260, 136)]


@pytest.mark.parametrize("case", range(len(FAR)))
@pytest.mark.parametrize("sx,sw,sy", [(-120, 100, -118), (100, -122, -119), (-124, 0, 60), (10, -118, -121), (-132, 90, -90), (90, 3, -133), (100, 3, 20), (112, -2, 10)])
def test_grouped_float32_keeps_its_accuracy_for_small_and_large_values(case, sx, sw, sy):
    """Rows, weights or gradients near and below the smallest normal float32, next to ones that bring the products back, and ones
    next to the largest: the bound of every other float32 product (the module's tolerances), and the last step of a subnormal result."""
    from weather_model_amd import ops
    sizes, N, K = FAR[case]
    M, G = sum(sizes), len(sizes)
    x, w, gy = (rows(case + k, s, torch.float32) * 2.0 ** e for k, s, e in ((1, (M, K), sx), (2, (G, N, K), sw), (3, (M, N), sy)))
    off = offsets_of(sizes)
    y = ops.dense_grouped_forward(x.cuda(), w.cuda(), off)
    gx, gw, _ = ops.dense_grouped_backward(x.cuda(), w.cuda(), off, gy.cuda(), need_bias=False)

    def near(got, ref, S, n, what):
        # a product or a partial sum below 2^-126 is rounded to 2^-149: half a step for each of n
        acc = (5 * (1.5 * n + 16) ** 0.5 * U + 3 * 2.0 ** -26) * S + (1.5 * n + 16) * 2.0 ** -150
        got, most = got.cpu().double(), torch.finfo(torch.float32).max
        d = (got - ref).abs()
        # past the largest float32 a sum is infinite; where S passes it, a partial sum may be, by the order of the sum
        beyond = ref.abs() > most * (1 + U) + acc
        assert not bool(got[beyond].isfinite().any()), what
        fine = (d <= (1 + U) * acc + U * ref.abs()) | ((S > most) & ~got.isfinite())
        assert bool(fine.all()), (what, float((d / S.clamp(min=1e-300)).max()))
    ref, S = grouped_ref(x, w, None, sizes, 0, False)
    near(y, ref, S, K, "y")
    ref, S = grouped_ref(gy, w.transpose(1, 2), None, sizes, 0, False)
    near(gx, ref, S, N, "gx")
    at = 0
    for g, n in enumerate(sizes):
        a, c = gy[at:at + n].double(), x[at:at + n].double()
        near(gw[g], a.t() @ c, a.abs().t() @ c.abs(), n, (g, "gw"))
        at += n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[9, 0, 4], [150, 0, 261], [1]])
def test_grouped_autograd_with_the_relu_masks_of_neighbours(sizes, dtype):
    """Two layers whose ReLU between them is masked by the upper one's gradient of rows (relu_bwd_fused below, relu_input above)
    give the gradients of the layers by themselves, bit for bit, and those of the formula in float64."""
    from weather_model_amd import ops
    M, G, K, H, N = sum(sizes) + 2, len(sizes), 40, 72, 33
    off = offsets_of(sizes)
    host = [rows(k, s, dtype, c) for k, s, c in ((1, (M, K), 1.0), (2, (G, H, K), K ** -0.5), (3, (G, H), 0.3), (4, (G, N, H), H ** -0.5), (5, (G, N), 0.3))]
    gout = rows(6, (M, N), dtype)

    def grads(below, above):
        x, w1, b1, w2, b2 = leaves = [t.cuda().requires_grad_() for t in host]
        h = ops.dense_grouped(x, w1, off, b1, relu=True, relu_bwd_fused=below)
        y = ops.dense_grouped(h, w2, off, b2, relu_input=above)
        y.backward(gout.cuda())
        return h.detach().cpu(), [t.grad for t in leaves]
    h, alone = grads(False, False)
    for below, above in ((True, True), (False, True)):       # masked twice is masked once
        h2, fused = grads(below, above)
        assert torch.equal(h, h2)
        for k, (a, b) in enumerate(zip(alone, fused)):
            assert torch.equal(a, b), (below, above, k)
    _, unmasked = grads(True, False)
    assert sum(sizes) < 2 or not torch.equal(unmasked[0], alone[0])
    # gh is rounded to the type once; what it is off by goes on into the lower layer's gradients
    half, tiny, at = half_step(dtype), torch.finfo(dtype).tiny, 0
    for g, n in enumerate(sizes):
        p = slice(at, at + n)
        go, hd, xd, w1, w2 = (t.double() for t in (gout[p], h[p], host[0][p], host[1][g], host[3][g]))
        mask = (hd > 0).double()
        gh, Sh = go @ w2 * mask, go.abs() @ w2.abs() * mask
        eh = 6 * (1.5 * N + 16) ** 0.5 * U * Sh + half * gh.abs() + tiny
        for what, got, ref, S, e, terms in (
                ("gw2", alone[3][g], go.t() @ hd, go.abs().t() @ hd, 0.0, n), ("gb2", alone[4][g], go.sum(0), go.abs().sum(0), 0.0, n),
                ("gw1", alone[1][g], gh.t() @ xd, gh.abs().t() @ xd.abs(), eh.t() @ xd.abs(), n), ("gb1", alone[2][g], gh.sum(0), gh.abs().sum(0), eh.sum(0), n),
                ("gx", alone[0][p], gh @ w1, gh.abs() @ w1.abs(), eh @ w1.abs(), H)):
            tol = 1.01 * (6 * (1.5 * terms + 16) ** 0.5 * U * (S + e) + e + half * (ref.abs() + e) + tiny)
            assert bool(((got.cpu().double() - ref).abs() <= tol).all()), (what, g)
        at += n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,p,offset", [(1, 0.5, 0), (4099, 0.1, 1), (100003, 0.9, 2), (65536, 0.5, 2 ** 33 + 3), (262144, 2.0 ** -16, 8), (5000, 1.0, 0)])
def test_dropout_zeros_are_the_dropped_elements_and_the_gradient_is_the_draws(n, p, offset, dtype):
    """Every type: a result is zero where and only where the element is dropped or was zero (a kept value grows), and the backward
    pass gives gy / (1 - p) of the same elements."""
    from weather_model_amd import ops
    x, gy = rows(n, (n,), dtype), rows(n + 1, (n,), dtype)
    x[:: 97], gy[:: 89] = torch.finfo(dtype).smallest_normal, -torch.finfo(dtype).smallest_normal
    keep = kept(n, p, 31, offset)
    scale = 0.0 if p == 1.0 else 1.0 / (1.0 - round(p * 2 ** 32) / 2 ** 32)
    for t, got in ((x, ops.dropout_forward(x.cuda(), p, 31, offset=offset)), (gy, ops.dropout_backward(gy.cuda(), p, 31, offset=offset))):
        got, ref = got.cpu(), torch.where(keep, t.double() * scale, 0.0)
        assert torch.equal(got == 0, ~keep | (t == 0))
        # the scale and the product are rounded in float32, the result to its type (a subnormal one to its last step)
        last = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert bool(((got.double() - ref).abs() <= (2.1 * U + half_step(dtype)) * ref.abs() + last / 2).all())
