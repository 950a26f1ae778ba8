"""4-bit weight products against the definition in 64 bits.

Tolerance of an output: half a step of its type (2^-11 relative for FP16, and
2^-25 absolute below the normals), plus the FP32 sums: with A = sum_k s (c + z)
|x| the magnitude that passes through them, each of the chained additions
off by at most 2^-23 of it: at most 20 at the end of a group and of the sum, one
for every column block, and 4 matrix instructions of a group, each of which
aligns 16 products and its sum so far to the largest and cuts them off there, 17
times 2^-23.  Bias and residual add a rounding each.
"""
import numpy as np
import pytest
import torch

from gpu_util import stream
from mruntime_b200 import capi

pytestmark = pytest.mark.gpu


def make(N, K, group, zeros, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8)
    scales = (0.001 + 0.02 * torch.rand(N, K // group, generator=g)).half()
    z = torch.randint(0, 16, (N, K // group), generator=g, dtype=torch.uint8) if zeros else None
    c = torch.stack((codes & 15, codes >> 4), -1).view(N, K).double()
    zz = z.double() if zeros else torch.full((N, K // group), 8.0, dtype=torch.float64)
    s, zz = (t.double().repeat_interleave(group, 1) for t in (scales, zz))
    d = [t.cuda() if t is not None else None for t in (codes, scales, z)]
    w = capi.WeightQ4.from_codes(d[0].data_ptr(), d[1].data_ptr(), capi.FP16, d[2].data_ptr() if zeros else None, True,
                                 N, K, group, stream())
    return w, s * (c - zz), s * (c + zz)


def bound(x, w, mag, out_eps, K):
    y = x.double() @ w.t()
    fp32 = (20 + 4 * 17 + K // 128 + 1) * 2.0 ** -23 * (x.double().abs() @ mag.t())
    return y, fp32 + out_eps * (y.abs() + fp32) + 2.0 ** -25


def run(w, x, **kw):
    xd = x.cuda()
    y = torch.full((x.shape[0], w.n), 7.0, dtype=torch.float32 if kw.get("y_dtype") == capi.FP32 else torch.float16,
                   device="cuda")
    capi.gemv_q4(w, xd.data_ptr(), x.shape[1], y.data_ptr(), w.n, x.shape[0], stream=stream(), **kw)
    capi.sync(stream())
    return y.cpu()


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 40])
@pytest.mark.parametrize("N,K,group,zeros", [(16, 128, 128, False), (5, 32, 32, True), (33, 96, 32, False),
                                             (200, 896, 64, True), (1152, 896, 128, False), (77, 4864, 32, True),
                                             (130, 192, 64, False), (24, 18944, 128, True)])
def test_product(cuda_dev, M, N, K, group, zeros):
    w, val, mag = make(N, K, group, zeros, M + N + K)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).half()
    x[0, K // 3] = 60.0
    y, tol = bound(x, val, mag, 2.0 ** -11, K)
    got = run(w, x)
    assert ((got.double() - y).abs() <= tol).all()
    y32, tol = bound(x, val, mag, 2.0 ** -24, K)
    assert ((run(w, x, y_dtype=capi.FP32).double() - y32).abs() <= tol).all()
    assert torch.equal(run(w, x), got)


@pytest.mark.parametrize("M,N,K,group,zeros", [(7, 700, 18944, 32, True), (16, 700, 18944, 128, False),
                                               (10, 1200, 9600, 64, True), (1, 1700, 9600, 64, False),
                                               (4, 4608, 512, 64, True), (25, 900, 9600, 128, True)])
def test_long_sums_cut_into_slices(cuda_dev, M, N, K, group, zeros):
    """Where x is too much for one CTA, or the rows too few for the device."""
    w, val, mag = make(N, K, group, zeros, N)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(N)).half()
    y, tol = bound(x, val, mag, 2.0 ** -11, K)
    got = run(w, x)
    assert ((got.double() - y).abs() <= tol).all()
    assert torch.equal(run(w, x), got)


def make_large(N, K, group, zeros, seed):
    """make() for weights that are told by slices of rows: the weight, and its values and magnitudes of rows a..b."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8, device="cuda")
    scales = (0.001 + 0.02 * torch.rand(N, K // group, generator=g, device="cuda")).half()
    z = torch.randint(0, 16, (N, K // group), generator=g, dtype=torch.uint8, device="cuda") if zeros else None
    w = capi.WeightQ4.from_codes(codes.data_ptr(), scales.data_ptr(), capi.FP16, z.data_ptr() if zeros else None, True,
                                 N, K, group, stream())

    def values(a, b):
        c = torch.stack((codes[a:b] & 15, codes[a:b] >> 4), -1).view(-1, K // group, group).double()
        s = scales[a:b].double()[:, :, None]
        zz = z[a:b].double()[:, :, None] if zeros else 8.0
        return (s * (c - zz)).view(-1, K), (s * (c + zz)).view(-1, K)

    return w, values


def check_large(w, values, x, got, out_eps, added=0.0):
    """Every output against 64-bit sums, a slice of rows at a time; `added`: to the product, once it is rounded."""
    step = max(16, (1 << 27) // w.k)
    xd = x.cuda()
    for a in range(0, w.n, step):
        val, mag = values(a, min(a + step, w.n))
        y, tol = bound(xd, val, mag, out_eps, w.k)
        extra = added[:, a:a + step].double().cuda() if torch.is_tensor(added) else 0.0
        tol = tol + (2.0 ** -11 * ((y + extra).abs() + tol) if torch.is_tensor(added) else 0.0)
        assert ((got[:, a:a + step].cuda().double() - y - extra).abs() <= tol).all(), f"rows from {a} on"


# No launch takes all of these: x is too long for a CTA without slices of K, and clusters have too few warps for the rows.
@pytest.mark.parametrize("N,K,group,zeros,Ms", [(28771, 18944, 32, True, (5, 7, 16)), (6100, 131072, 128, False, (4, 9)),
                                                (32000, 98304, 128, True, (1, 3))])
def test_long_rows_of_large_weights(cuda_dev, N, K, group, zeros, Ms):
    w, values = make_large(N, K, group, zeros, K)
    for M in Ms:
        g = torch.Generator().manual_seed(M)
        x = torch.randn(M, K, generator=g).half()
        got = run(w, x)
        check_large(w, values, x, got, 2.0 ** -11)
        assert torch.equal(run(w, x), got)
        check_large(w, values, x, run(w, x, y_dtype=capi.FP32), 2.0 ** -24)
        res = torch.randn(M, N, generator=g).half()
        rd = res.cuda()
        check_large(w, values, x, run(w, x, res_ptr=rd.data_ptr(), ldr=N), 2.0 ** -11, res)


# Stretches of several tiles a warp, with a piece of a tile at each end; the last CTA short, the last tile not whole.
@pytest.mark.parametrize("N,K,group,zeros", [(152064, 3584, 128, False), (152057, 3584, 64, True), (150003, 512, 64, True),
                                             (149993, 640, 32, False), (60010, 896, 128, True)])
@pytest.mark.parametrize("M", [1, 7, 16])
def test_warps_with_many_tiles(cuda_dev, N, K, group, zeros, M):
    w, values = make_large(N, K, group, zeros, N + M)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).half()
    got = run(w, x)
    check_large(w, values, x, got, 2.0 ** -11)
    assert torch.equal(run(w, x), got)
    check_large(w, values, x, run(w, x, y_dtype=capi.FP32), 2.0 ** -24)


@pytest.mark.parametrize("M", [14, 30])
def test_fewer_tokens_at_a_time_where_more_have_no_plan(cuda_dev, M):
    w, values = make_large(28771, 18944, 32, True, M)
    x = torch.randn(M, 18944, generator=torch.Generator().manual_seed(M)).half()
    check_large(w, values, x, run(w, x), 2.0 ** -11)


def test_bias_of_a_weight_in_parts(cuda_dev):
    N, K = 6100, 131072
    w, values = make_large(N, K, 128, False, 3)
    b = torch.randn(N, generator=torch.Generator().manual_seed(1)).half()
    bd = b.cuda()
    w.attach_bias(bd.data_ptr(), capi.FP16, True, stream())
    x = torch.randn(4, K, generator=torch.Generator().manual_seed(2)).half()
    check_large(w, values, x, run(w, x, bias=True), 2.0 ** -11, b[None].expand(4, N))


def test_k_beyond_shared_memory_is_refused(cuda_dev):
    K = 1 << 20
    w = make_large(16, K, 128, False, 1)[0]
    t = torch.zeros(K, dtype=torch.float16, device="cuda")
    assert capi.lib().mrt_gemv_q4(w.h, t.data_ptr(), K, None, 0, t.data_ptr(), 0, 16, 1, 0, stream()) == 2
    capi.sync(stream())


def test_one_weight_on_two_streams(cuda_dev):
    """Calls that overlap give what they give alone."""
    w, _, _ = make(700, 4096, 64, True, 4)
    xs = [torch.randn(m, 4096, generator=torch.Generator().manual_seed(m)).half() for m in (1, 16)]
    want = [run(w, x) for x in xs]
    xd, streams = [x.cuda() for x in xs], [torch.cuda.Stream() for _ in xs]
    ys = [torch.zeros(8, x.shape[0], 700, dtype=torch.float16, device="cuda") for x in xs]
    torch.cuda.synchronize()
    for i in range(8):
        for x, y, s in zip(xd, ys, streams):
            capi.gemv_q4(w, x.data_ptr(), 4096, y[i].data_ptr(), 700, x.shape[0], stream=s.cuda_stream)
    torch.cuda.synchronize()
    capi.sync(stream())
    for y, o in zip(ys, want):
        assert (y.cpu() == o).all()


@pytest.mark.parametrize("M", [1, 5, 20])
def test_bias_and_residual(cuda_dev, M):
    N, K = 90, 256
    w, val, mag = make(N, K, 64, True, M)
    g = torch.Generator().manual_seed(9)
    x, b, res = torch.randn(M, K, generator=g).half(), torch.randn(N, generator=g).bfloat16(), torch.randn(M, N, generator=g).half()
    bd = b.cuda()
    w.attach_bias(bd.data_ptr(), capi.BF16, True, stream())
    y, tol = bound(x, val, mag, 2.0 ** -11, K)
    y1 = y + b.half().double()
    tol1 = tol + 2.0 ** -11 * (y1.abs() + tol)
    assert ((run(w, x, bias=True).double() - y1).abs() <= tol1).all()
    y2 = y1 + res.double()
    tol2 = tol1 + 2.0 ** -11 * (y2.abs() + tol1)
    rd = res.cuda()
    assert ((run(w, x, bias=True, res_ptr=rd.data_ptr(), ldr=N).double() - y2).abs() <= tol2).all()
    xd = x.cuda()  # in place: y is the residual
    capi.gemv_q4(w, xd.data_ptr(), K, rd.data_ptr(), N, M, bias=True, res_ptr=rd.data_ptr(), ldr=N, stream=stream())
    capi.sync(stream())
    assert ((rd.cpu().double() - y2).abs() <= tol2).all()


@pytest.mark.parametrize("off,ldx,ldy", [(0, 256, 50), (1, 257, 51), (4, 260, 64), (8, 264, 50)])
def test_strides_and_alignment(cuda_dev, off, ldx, ldy):
    N, K, M = 50, 256, 3
    w, val, mag = make(N, K, 32, False, off)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(off)).half()
    buf = torch.zeros(off + M * ldx, dtype=torch.float16, device="cuda")
    for m in range(M):
        buf[off + m * ldx:off + m * ldx + K] = x[m].cuda()
    out = torch.full((M, ldy), 3.0, dtype=torch.float16, device="cuda")
    capi.gemv_q4(w, buf.data_ptr() + 2 * off, ldx, out.data_ptr(), ldy, M, stream=stream())
    capi.sync(stream())
    y, tol = bound(x, val, mag, 2.0 ** -11, K)
    assert ((out[:, :N].cpu().double() - y).abs() <= tol).all()
    assert (out[:, N:] == 3.0).all()


def test_a_token_does_not_touch_another(cuda_dev):
    N, K, M = 40, 512, 9
    w, val, mag = make(N, K, 128, True, 3)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(3)).half()
    want = run(w, x)
    x[2, 17], x[8, 100] = float("nan"), float("inf")
    got = run(w, x)
    keep = [m for m in range(M) if m not in (2, 8)]
    assert torch.equal(got[keep], want[keep])
    assert not torch.isfinite(got[[2, 8]]).any()


@pytest.mark.parametrize("dt", [capi.FP16, capi.BF16, capi.FP32])
@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("on_device", [False, True])
def test_upload_rounds_to_nearest(cuda_dev, dt, symmetric, on_device):
    N, K, group = 37, 192, 64
    t = {capi.FP16: torch.float16, capi.BF16: torch.bfloat16, capi.FP32: torch.float32}[dt]
    src = (torch.randn(N, K, generator=torch.Generator().manual_seed(5)) * 0.05).to(t)
    src[3, :64] = 0
    src[4, 64:128] = src[4, 64:128].abs()
    src = src.cuda() if on_device else src
    w = capi.WeightQ4(src.data_ptr(), dt, on_device, N, K, group, symmetric, stream())
    out = torch.empty(N, K, dtype=torch.float16, device="cuda")
    w.read(out.data_ptr(), stream=stream())
    capi.sync(stream())
    v = src.cpu().double().view(N, -1, group)
    if symmetric:
        step = v.abs().amax(-1, keepdim=True) / 7
    else:
        step = (v.amax(-1, keepdim=True).clamp(min=0) - v.amin(-1, keepdim=True).clamp(max=0)) / 15
    # half a step, the scale's own rounding at the far end of the range, the rounding of the value read
    tol = step * (0.5 + 15 * 2.0 ** -11) + 2.0 ** -11 * v.abs() + 16 * 2.0 ** -24
    assert ((out.cpu().double().view(N, -1, group) - v).abs() <= tol).all()
    assert (out[3, :64] == 0).all()


def test_read_gives_the_held_values(cuda_dev):
    w, val, _ = make(45, 160, 32, True, 8)
    out = torch.full((45, 170), 5.0, dtype=torch.float16, device="cuda")
    w.read(out.data_ptr(), 170, stream())
    capi.sync(stream())
    assert torch.equal(out[:, :160].cpu(), val.half()) and (out[:, 160:] == 5.0).all()


def test_captured_chain_on_a_side_stream(cuda_dev):
    """Two products in a row, the second on the first's output, captured once and replayed on new x."""
    w1, v1, _ = make(256, 128, 32, True, 1)
    w2, v2, _ = make(64, 256, 64, False, 2)
    s = torch.cuda.Stream()
    x = torch.zeros(2, 128, dtype=torch.float16, device="cuda")
    h, y = (torch.zeros(2, n, dtype=torch.float16, device="cuda") for n in (256, 64))

    def step(st):
        capi.gemv_q4(w1, x.data_ptr(), 128, h.data_ptr(), 256, 2, stream=st)
        capi.gemv_q4(w2, h.data_ptr(), 256, y.data_ptr(), 64, 2, stream=st)

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(torch.cuda.current_stream().cuda_stream)
    for seed in range(3):
        new = torch.randn(2, 128, generator=torch.Generator().manual_seed(seed)).half()
        x.copy_(new.cuda())
        g.replay()
        torch.cuda.synchronize()
        got = y.cpu()
        step(stream())
        capi.sync(stream())
        assert torch.equal(got, y.cpu())
        assert torch.isfinite(got).all() and got.abs().sum() > 0


def test_refusals(cuda_dev):
    w, _, _ = make(32, 64, 32, False, 1)
    t = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    p = t.data_ptr()

    def code(**kw):
        a = dict(w=w.h, x=p, ldx=64, res=None, ldr=0, y=p, dt=0, ldy=32, M=1, flags=0)
        a.update(kw)
        return capi.lib().mrt_gemv_q4(a["w"], a["x"], a["ldx"], a["res"], a["ldr"], a["y"], a["dt"], a["ldy"], a["M"],
                                      a["flags"], stream())

    assert code(M=0) == 0
    assert code(M=-1) == 2 and code(ldx=63) == 2 and code(ldy=31) == 2 and code(res=p, ldr=31) == 2
    assert code(x=None) == 1 and code(y=None) == 1 and code(flags=2) == 1
    assert code(flags=1) == 1  # no bias attached
    assert code(dt=1) == 3 and code(dt=7) == 3
    assert code(dt=2, res=p, ldr=32) == 7
    with pytest.raises(capi.MrtError):
        w.read(p, 63, stream())
    capi.sync(stream())
