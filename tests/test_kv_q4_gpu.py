"""The paged 4-bit cache: append with rotation, read, attention, against their
definitions in 64 bits."""
import math

import pytest
import torch

from gpu_util import stream
from mruntime_b200 import capi

pytestmark = pytest.mark.gpu

DT = {torch.float16: capi.FP16, torch.bfloat16: capi.BF16}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Cache:
    """A cache of some sequences (new tokens, held tokens), its pages in no order among others' pages."""

    def __init__(self, lens, heads, kv_heads, D, page=16, theta=0.0, seed=0, spare=3, extra_rows=0, pages=None):
        g = torch.Generator().manual_seed(seed + 100)
        self.lens, self.H, self.Hk, self.D, self.page = lens, heads, kv_heads, D, page
        per = [-(-kv // page) for _, kv in lens]
        n = pages or sum(per) + spare
        order = torch.randperm(n, generator=g).to(torch.int32)
        self.ld = max(per + [1]) + 1
        table = torch.full((len(lens), self.ld), -1, dtype=torch.int32)  # what is not needed is no page
        at = 0
        for b, k in enumerate(per):
            table[b, :k] = order[at:at + k]
            at += k
        self.table = table.cuda()
        self.kv = capi.KvQ4(n, page, kv_heads, D, theta)
        self.T = sum(q for q, _ in lens) + extra_rows
        self.batch = self.make_batch([q for q, _ in lens], self.T)

    def make_batch(self, new, tokens=None, held=None, **kw):
        start = torch.tensor([0] + list(new)).cumsum(0).to(torch.int32).cuda()
        kv = torch.tensor(held if held is not None else [k for _, k in self.lens], dtype=torch.int32).cuda()
        b = capi.KvBatch(len(new), int(start[-1]) if tokens is None else tokens, kw.get("max_q", max(list(new) + [0])),
                         kw.get("max_kv", max([k for _, k in self.lens] + [0])), start.data_ptr(), kv.data_ptr(),
                         self.table.data_ptr(), self.ld)
        b.keep = (start, kv)
        return b

    def append(self, batch, k, v, q=None, q_out=None, st=None):
        H = 0 if q is None else self.H
        self.kv.append(batch, DT[k.dtype], q.data_ptr() if H else None, H * self.D, H, q_out.data_ptr() if H else None,
                       H * self.D, k.data_ptr(), self.Hk * self.D, v.data_ptr(), self.Hk * self.D, st or stream())

    def fill(self, k, v):
        """Every held token of every sequence, sequences one after another."""
        self.append(self.make_batch([kv for _, kv in self.lens]), k, v)
        capi.sync(stream())

    def read(self, batch, dtype=torch.float16):
        k = torch.full((batch.tokens, self.Hk, self.D), 9.0, dtype=dtype, device="cuda")
        v = torch.full_like(k, 9.0)
        self.kv.read(batch, DT[dtype], k.data_ptr(), self.Hk * self.D, v.data_ptr(), self.Hk * self.D, stream())
        capi.sync(stream())
        return k.cpu(), v.cpu()

    def attend(self, q, causal, scale=None, batch=None, out=None, st=None, ws=None):
        batch = batch or self.batch
        out = torch.full_like(q, 9.0) if out is None else out
        if ws is None:
            n = self.kv.attention_workspace(batch, self.H)
            ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")  # nothing is expected of it
        self.kv.attention(batch, DT[q.dtype], q.data_ptr(), self.H * self.D, self.H, out.data_ptr(), self.H * self.D,
                          scale or self.D ** -0.5, causal, ws.data_ptr(), ws.numel(), st or stream())
        return out


def quantised(x):
    """The held values of rows of FP32 x, in 64 bits, by the definition's own FP32 steps."""
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    s = ((hi - lo) * torch.tensor(1.0 / 15.0)).half().float().clamp(min=2.0 ** -24)
    inv = 1.0 / s
    z = torch.round(-lo * inv).clamp(0, 15)
    c = (torch.round(x * inv) + z).clamp(0, 15)
    return (c - z).double() * s.double(), s.double()


def rows(g, *shape, dtype=torch.float16, spread=1.0):
    x = torch.randn(*shape, generator=g) * spread
    x[..., 3] += 3.0
    return x.to(dtype)


def rotated(x, pos, theta):
    half = x.shape[-1] // 2
    a = pos.double()[:, None] * torch.tensor([float(theta) ** (-i / half) for i in range(half)], dtype=torch.float64)
    c, s = a.cos()[:, None], a.sin()[:, None]
    x0, x1 = x.double()[..., :half], x.double()[..., half:]
    return torch.cat((x0 * c - x1 * s, x0 * s + x1 * c), -1)


LENS = [(1, 1), (3, 17), (16, 16), (1, 200), (0, 5), (33, 40), (0, 0), (2, 64)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page", [16, 48, 128])
@pytest.mark.parametrize("theta", [0.0, 10000.0, 1000000.0])
def test_append(cuda_dev, D, dtype, page, theta):
    c = Cache(LENS, 6, 3, D, page, theta, seed=page, extra_rows=2)
    g = torch.Generator().manual_seed(D)
    q, k, v = (rows(g, c.T, h, D, dtype=dtype) for h in (6, 3, 3))
    k[1, 1] = 0  # a row of zeros
    v[2, 0] = v[2, 0].abs()  # a range that ends at zero
    qo = torch.full_like(q, 9.0).cuda()
    c.append(c.batch, k.cuda(), v.cuda(), q.cuda(), qo)
    kr, vr = c.read(c.batch)
    n = c.T - 2
    pos = torch.cat([torch.arange(kv - m, kv) for m, kv in LENS])
    if theta:
        qx, kx = rotated(q[:n], pos, theta), rotated(k[:n], pos, theta)
    else:
        qx, kx = q[:n].double(), k[:n].double()
    # cos and sin to half a step, two products and a sum in FP32, then the output's own step
    size = lambda x: x.double().square().view(*x.shape[:2], 2, -1).sum(2, keepdim=True).sqrt().expand(-1, -1, 2, -1).reshape(x.shape)  # noqa: E731
    tol = HALF_STEP[dtype] * qx.abs() + 2.0 ** -21 * size(q[:n]) + 2.0 ** -25
    assert ((qo[:n].cpu().double() - qx).abs() <= tol).all()
    for x, got in ((kx, kr[:n]), (v[:n].double(), vr[:n])):
        step = ((x.amax(-1).clamp(min=0) - x.amin(-1).clamp(max=0)) / 15)[..., None]
        # half a step, the scale's rounding over the range, FP32's, the rounding of the value read
        tol = step * (0.5 + 15 * 2.0 ** -11 + 2.0 ** -12) + 2.0 ** -11 * x.abs() + 16 * 2.0 ** -24
        assert ((got.double() - x).abs() <= tol).all()
    # the codes themselves: V's are those of the definition's own steps, exactly
    want, _ = quantised(v[:n].float())
    assert torch.equal(vr[:n], want.half())
    if not theta:
        assert torch.equal(kr[:n], quantised(k[:n].float())[0].half())
    for t in (qo.cpu(), kr, vr):
        assert (t[n:] == 9.0).all()  # rows behind the last sequence


def test_append_leaves_other_tokens_alone(cuda_dev):
    """Token by token and all at once give the same cache; a page's other half and other pages stay."""
    lens = [(40, 40), (25, 25)]
    g = torch.Generator().manual_seed(4)
    k, v = rows(g, 65, 2, 64).cuda(), rows(g, 65, 2, 64).cuda()
    a, b = (Cache(lens, 2, 2, 64, 32, 10000.0, seed=1) for _ in range(2))
    a.fill(k, v)
    for t in range(40):
        new = [1, 1 if t < 25 else 0]
        at = [t, 40 + t]
        rowsel = at[:1 + new[1]]
        b.append(b.make_batch(new, held=[t + 1, min(t + 1, 25)]), k[rowsel].contiguous(), v[rowsel].contiguous())
        capi.sync(stream())
    whole = a.make_batch([40, 25])
    for x, y in zip(a.read(whole), b.read(whole)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("pos", [0, 1, 131071, 1000003, 2 ** 31 - 1000])
def test_rotation_at_far_positions(cuda_dev, pos):
    """The angle is exact at any position: the table row only has to name the page that is written."""
    D, theta = 128, 10000.0
    page = 1 << 20
    kv = capi.KvQ4(1, page, 1, D, theta)
    g = torch.Generator().manual_seed(1)
    q, k = rows(g, 1, 2, D), rows(g, 1, 1, D)
    n = pos // page + 1
    table = torch.zeros(1, n, dtype=torch.int32, device="cuda")
    start, held = torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.tensor([pos + 1], dtype=torch.int32, device="cuda")
    b = capi.KvBatch(1, 1, 1, pos + 1, start.data_ptr(), held.data_ptr(), table.data_ptr(), n)
    qd, kd = q.cuda(), k.cuda()
    kv.append(b, capi.FP16, qd.data_ptr(), 2 * D, 2, qd.data_ptr(), 2 * D, kd.data_ptr(), D, kd.data_ptr(), D, stream())
    capi.sync(stream())
    import numpy as np
    from decimal import Decimal, getcontext

    getcontext().prec = 60
    two_pi = Decimal("6.28318530717958647692528676655900576839433879875021164194988918461563281257")
    turns = [(Decimal(pos) * (Decimal(10000) ** (Decimal(-2 * i) / Decimal(D))) / two_pi) % 1 for i in range(D // 2)]
    a = np.array([float(t * two_pi) for t in turns])
    x = q.double().numpy()[0]
    c, s = np.cos(a), np.sin(a)
    want = np.concatenate((x[:, :64] * c - x[:, 64:] * s, x[:, :64] * s + x[:, 64:] * c), -1)
    size = np.sqrt(x[:, :64] ** 2 + x[:, 64:] ** 2)
    tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -21 * np.concatenate((size, size), -1) + 2.0 ** -25
    assert (np.abs(qd.cpu().double().numpy()[0] - want) <= tol).all()


@pytest.mark.parametrize("ldq,off", [(0, 0), (3, 1), (8, 4)])
def test_append_strides_in_place(cuda_dev, ldq, off):
    """q, k and v as slices of one product's rows, at any alignment; q rotated in place."""
    H, Hk, D, theta, lens = 4, 2, 64, 10000.0, [(5, 9), (2, 2)]
    c, d = (Cache(lens, H, Hk, D, 16, theta, seed=2) for _ in range(2))
    g = torch.Generator().manual_seed(3)
    q, k, v = rows(g, 7, H, D), rows(g, 7, Hk, D), rows(g, 7, Hk, D)
    qo = torch.empty_like(q).cuda()
    c.append(c.batch, k.cuda(), v.cuda(), q.cuda(), qo)
    ld = (H + 2 * Hk) * D + ldq
    buf = torch.full((off + 7 * ld,), 9.0, dtype=torch.float16, device="cuda")
    view = buf[off:].view(7, ld)
    view[:, :H * D], view[:, H * D:(H + Hk) * D], view[:, (H + Hk) * D:(H + 2 * Hk) * D] = (
        t.reshape(7, -1).cuda() for t in (q, k, v))
    p = buf.data_ptr() + 2 * off
    d.kv.append(d.batch, capi.FP16, p, ld, H, p, ld, p + 2 * H * D, ld, p + 2 * (H + Hk) * D, ld, stream())
    capi.sync(stream())
    assert torch.equal(view[:, :H * D].reshape(7, H, D), qo)
    assert torch.equal(view[:, H * D:(H + Hk) * D].cpu(), k.reshape(7, -1)) and (view[:, (H + 2 * Hk) * D:] == 9.0).all()
    for x, y in zip(c.read(c.batch), d.read(d.batch)):
        assert torch.equal(x, y)


# (lowest, highest) channel of rows whose codes could mean more than FP16 holds
WIDE = [(-2000.0, 65504.0), (-60000.0, 65504.0), (-65504.0, 60000.0), (-60000.0, 63000.0), (0.0, 65504.0),
        (-65504.0, 0.0), (-65504.0, 65504.0), (-500.0, 65504.0)]


def wide_rows(n, heads, D, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.zeros(n, heads, D)
    for i in range(n):
        lo, hi = WIDE[i % len(WIDE)]
        x[i] = lo + (hi - lo) * torch.rand(heads, D, generator=g)
        x[i, :, i % D], x[i, :, (i + 7) % D] = lo, hi
    return x.half()


def held_finite(x):
    """quantised() with the scale lowered until every code's value is a finite FP16."""
    lo, hi = x.amin(-1, keepdim=True).clamp(max=0), x.amax(-1, keepdim=True).clamp(min=0)
    s = ((hi - lo) * torch.tensor(1.0 / 15.0)).half().float().clamp(min=2.0 ** -24)
    z = torch.round(-lo * (1.0 / s)).clamp(0, 15)
    most = torch.maximum(z, 15 - z)
    low = (65504.0 / most).half()  # the largest FP16 below: one less where this rounded up
    low = torch.where(low.double() * most.double() > 65504, torch.nextafter(low, torch.zeros_like(low)), low).float()
    s = torch.where(s * most > 65504, low, s)
    c = (torch.round(x * (1.0 / s)) + z).clamp(0, 15)
    return (c - z).double() * s.double(), s.double()


def test_wide_rows_in_the_oracle_are_finite_and_near():
    x = wide_rows(64, 2, 64, 1).float()
    v, _ = held_finite(x)
    assert float(v.abs().max()) <= 65504
    # In steps s before it is lowered, to s': the near end n = 15 - z steps away, n s > 65504 >= hi, n >= 8 > z (s < 8736).
    # The far end is off by z's rounding, 1/2, and z (s - s').  n s - hi = n s - range - lo <= (1/2 + 15 2^-11) s, as
    # range >= 15 s (1 - 2^-11) and -lo <= (z + 1/2) s; s' is FP16, 2^-10 of itself less at most; z / n <= 7 / 8.
    old, s = quantised(x)
    assert ((v - x).abs() / s).max() <= 0.5 + 7 / 8 * (0.5 + 15 * 2.0 ** -11) + 7 * 2.0 ** -10
    assert float(old.abs().max()) > 65520  # without it they are not


@pytest.mark.parametrize("D", [64, 128])
def test_wide_rows_are_held_in_fp16(cuda_dev, D):
    """Magnitudes up to 65504 are taken; what they read back as is finite and within a step."""
    c = Cache([(40, 40)], 2, 2, D, 16, seed=2)
    k, v = wide_rows(40, 2, D, 1), wide_rows(40, 2, D, 2)
    c.append(c.batch, k.cuda(), v.cuda())
    for x, got in zip((k, v), c.read(c.batch)):
        assert torch.isfinite(got).all()
        assert torch.equal(got, held_finite(x.float())[0].half())


@pytest.mark.parametrize("n,kv", [(3, 40), (140, 150)])
def test_wide_values_reach_no_row_that_does_not_see_them(cuda_dev, n, kv):
    """Values near the largest FP16 at a position that earlier rows do not see, and in the last page's tail where
    an earlier owner left them."""
    H, Hk, D = 4, 2, 64
    c = Cache([(n, kv)], H, Hk, D, 16, seed=1)
    q, k, v = held_rows(c, 2)
    c.fill(k.cuda(), v.cuda())
    clean = c.attend(q.cuda(), True)
    capi.sync(stream())
    tail = -(-kv // 16) * 16
    assert tail > kv
    t = Cache([(tail, tail)], H, Hk, D, 16, seed=1)
    t.kv, t.table, t.ld = c.kv, c.table, c.ld
    wide = wide_rows(tail, Hk, D, 5).cuda()
    t.fill(wide, wide)
    c.fill(k.cuda(), v.cuda())
    out = c.attend(q.cuda(), True)
    capi.sync(stream())
    assert torch.equal(out, clean)
    v2 = v.clone()
    v2[kv - 2:] = wide[:2].cpu()
    c.fill(k.cuda(), v2.cuda())
    out = c.attend(q.cuda(), True)
    capi.sync(stream())
    sees = torch.arange(kv - n, kv) >= kv - 2
    assert torch.equal(out[~sees.cuda()], clean[~sees.cuda()])
    (kx, _), (vx, vs) = quantised(k.float()), held_finite(v2.float())
    want, tol = reference(c, q, kx, vx, vs, True, D ** -0.5)
    assert ((out.cpu().double() - want).abs() <= tol).all()


def test_non_finite_rows_read_back_as_nan(cuda_dev):
    c = Cache([(6, 6)], 1, 1, 128, 16)
    x = torch.ones(6, 1, 128, dtype=torch.bfloat16)
    x[1, 0, 5], x[2, 0, 127], x[3, 0, 0], x[4, 0, 9] = float("nan"), float("inf"), float("-inf"), 1e30
    c.append(c.batch, x.cuda(), x.cuda())
    for t in c.read(c.batch, torch.bfloat16):
        assert torch.isnan(t[1:5]).all() and (t[0] == 1).all() and (t[5] == 1).all()


# ------------------------------------------------------------------ attention

def reference(c, q, kx, vx, vs, causal, scale):
    """64-bit attention, and the tolerance of each output.

    Few rows (32 of a sequence and kv head): each probability times its value's
    scale is rounded to FP16, 2^-11 of it, or where it is small 2^-25 of the
    row's largest such product (codes up to 15).  Many rows: each probability
    is, by 2^-11 or 2^-25 of the row's largest, and each value, by 2^-11 or
    2^-25.  A
    score is off by FP32 sums of the products' magnitude (2^-23 for each of the
    chained additions: 17 in a matrix instruction, which aligns 16 products and
    its sum so far to the largest and cuts them off there, D / 16 of them) and its
    own size, and moves its probability by as much; the sums over keys are off by
    2^-23 for each of theirs (17 per 16 keys, and the joins); the output by half a
    step.
    Codes and zero points may be summed apart: s (c + z) <= |value| + 30 s, and a
    key's 30 s is at most 4 times its largest channel."""
    H, Hk, D = c.H, c.Hk, c.D
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    row = tok = 0
    many = max(n for n, _ in c.lens) * H // Hk > 32
    for n, kv in c.lens:
        k, v, sv = kx[tok:tok + kv].cuda(), vx[tok:tok + kv].cuda(), vs[tok:tok + kv].cuda()
        for i in range(n):
            keys = kv - n + i + 1 if causal else kv
            if keys <= 0:
                continue
            qd = q[row + i].double().cuda().view(Hk, H // Hk, D)
            s = torch.einsum("hgd,thd->hgt", qd, k[:keys]) * scale
            mag = torch.einsum("hgd,thd->hgt", qd.abs(), k[:keys].abs() + 4 * k[:keys].abs().amax(-1, keepdim=True)) * abs(scale)
            p = s.softmax(-1)
            o = torch.einsum("hgt,thd->hgd", p, v[:keys])
            off = (17 * D / 16 * 2.0 ** -23 * mag + 2.0 ** -22 * s.abs() + 2.0 ** -21)
            pv = torch.einsum("hgt,thd->hgd", p * (2.0 ** (-10 if many else -11) + 2 * off), v[:keys].abs())
            pv += (32 + 17 * keys / 16) * 2.0 ** -23 * torch.einsum("hgt,thd->hgd", p, v[:keys].abs() + 30 * sv[:keys])
            mean_off = (p * off).sum(-1, keepdim=True)
            if many:
                low = p.amax(-1, keepdim=True) * 2.0 ** -25 * v[:keys].abs().sum(0)[:, None] + 2.0 ** -25
            else:
                low = (p * sv[:keys].permute(1, 2, 0)).amax(-1, keepdim=True) * 2.0 ** -25 * 15 * keys
            out[row + i] = o.reshape(H, D).cpu()
            tol[row + i] = (pv + 2 * mean_off * o.abs() + low + HALF_STEP[q.dtype] * o.abs() + 2.0 ** -25).reshape(H, D).cpu()
        row, tok = row + n, tok + kv
    return out, tol


def held_rows(c, seed, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    total = sum(kv for _, kv in c.lens)
    k, v = rows(g, total, c.Hk, c.D, dtype=dtype), rows(g, total, c.Hk, c.D, dtype=dtype)
    v *= torch.exp(torch.randn(total, c.Hk, 1, generator=g)).to(dtype)  # values of unlike sizes
    q = torch.randn(c.T, c.H, c.D, generator=g).to(dtype)
    return q, k, v


ATTN = [
    ([(1, 1)], 2, 2, 64, 16), ([(1, 15), (1, 16), (1, 17), (1, 0), (1, 33)], 4, 1, 128, 16),
    ([(1, 517)], 14, 2, 64, 16), ([(1, 700), (1, 3), (1, 129)], 28, 4, 128, 64),
    ([(3, 3), (2, 40), (0, 9), (4, 300)], 7, 1, 64, 32), ([(5, 77), (1, 130)], 16, 1, 128, 16),
    ([(70, 70), (1, 200), (33, 140)], 12, 4, 128, 48), ([(130, 517)], 14, 2, 64, 16), ([(9, 5), (4, 4)], 6, 3, 64, 16),
    ([(300, 300), (2, 1000)], 2, 2, 128, 128), ([(1, 4099)], 8, 8, 64, 16), ([(1, 9000)], 40, 1, 128, 32),
    ([(150, 400), (129, 129)], 9, 3, 64, 16),
]


@pytest.mark.parametrize("case", range(len(ATTN)))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
def test_attention(cuda_dev, case, dtype, causal):
    lens, H, Hk, D, page = ATTN[case]
    c = Cache(lens, H, Hk, D, page, seed=case, extra_rows=1)
    q, k, v = held_rows(c, case, dtype)
    c.fill(k.cuda(), v.cuda())
    out = c.attend(q.cuda(), causal)
    capi.sync(stream())
    (kx, _), (vx, vs) = quantised(k.float()), quantised(v.float())
    want, tol = reference(c, q, kx, vx, vs, causal, D ** -0.5)
    n = c.T - 1
    bad = (out[:n].cpu().double() - want[:n]).abs() > tol[:n]
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst " \
        f"{float(((out[:n].cpu().double() - want[:n]).abs() / tol[:n].clamp(min=1e-30)).max()):.2f} of the tolerance"
    assert (out[n:] == 9.0).all()
    again = c.attend(q.cuda(), causal)
    capi.sync(stream())
    assert torch.equal(out, again)
    qd = q.cuda()
    c.attend(qd, causal, out=qd)  # in place
    capi.sync(stream())
    assert torch.equal(qd[:n], out[:n])


def attention64(c, q, kx, vx, causal, rounded=None):
    """64-bit attention of whole sequences; `rounded`: the type that probabilities (relative to their row's largest)
    and, of many rows, values are rounded to on the way."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    many = max(n for n, _ in c.lens) * c.H // c.Hk > 32
    row = tok = 0
    for n, kv in c.lens:
        s = torch.einsum("nhgd,thd->hgnt", q[row:row + n].double().view(n, c.Hk, -1, c.D), kx[tok:tok + kv]) * c.D ** -0.5
        if causal:
            s = s.masked_fill(torch.ones(n, kv, dtype=torch.bool).triu(kv - n + 1), -math.inf)
        p = (s - s.amax(-1, keepdim=True)).exp()
        w, v = p, vx[tok:tok + kv]
        if rounded is not None:
            w, v = p.to(rounded).double(), v.to(rounded).double() if many else v
        out[row:row + n] = torch.einsum("hgnt,thd->nhgd", w / p.sum(-1, keepdim=True), v).reshape(n, c.H, c.D)
        row, tok = row + n, tok + kv
    return out


@pytest.mark.parametrize("lens,H,Hk,D", [([(1, 517), (1, 1200), (1, 90)], 28, 4, 128), ([(1, 700), (1, 350)], 14, 2, 64),
                                         ([(3, 400), (2, 1500)], 28, 4, 128), ([(64, 300), (40, 700)], 14, 2, 64),
                                         ([(90, 500)], 28, 4, 128), ([(130, 130), (7, 900)], 12, 4, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_rounds_to_fp16_and_no_further(cuda_dev, lens, H, Hk, D, causal):
    """The error of a whole call.  Of numbers whose mantissas are spread evenly over the logarithm, rounding to FP16
    is off by 2^-11 sqrt(1/3 . 3/4 / (2 ln 2)) = 0.425 2^-11 in the root mean square.  There are three: of the outputs,
    and of probabilities and (of many rows) values, whose terms p v, of either sign, add up as their errors do; so
    sqrt(3) 0.425 = 0.74 of 2^-11 in all, FP32 sums being 2^-20 of it.  Rounded to BF16 instead, at 8 times that, the
    same inputs are beyond the bound."""
    c = Cache(lens, H, Hk, D, 16, seed=D + H)
    g = torch.Generator().manual_seed(H)
    total = sum(kv for _, kv in lens)
    q, k, v = (torch.randn(n, h, D, generator=g).half() for n, h in ((c.T, H), (total, Hk), (total, Hk)))
    c.fill(k.cuda(), v.cuda())
    out = c.attend(q.cuda(), causal)
    capi.sync(stream())
    kx, vx = quantised(k.float())[0], quantised(v.float())[0]
    want = attention64(c, q, kx, vx, causal)
    err = lambda x: float((x.double() - want).norm() / want.norm())  # noqa: E731
    assert err(attention64(c, q, kx, vx, causal, torch.float16).half()) <= 2.0 ** -11
    assert err(attention64(c, q, kx, vx, causal, torch.bfloat16).half()) > 2.0 ** -11
    assert err(out.cpu()) <= 2.0 ** -11


@pytest.mark.parametrize("lens,H,Hk,D", [([(300, 6000)], 28, 4, 128), ([(400, 2000), (30, 3000)], 14, 2, 64),
                                         ([(3, 800), (2, 900)] * 3, 4, 2, 64), ([(2, 1000)] * 40, 14, 2, 128)])
@pytest.mark.parametrize("ahead", [8.0, 14.0])
def test_a_first_key_that_takes_most_of_every_row(cuda_dev, lens, H, Hk, D, ahead):
    """Its value is next to nothing, so that the outputs are made of probabilities that are e^-8 and e^-14 of their row's
    largest.  e^-14 is 2^-20.2, and 2^-13.2 where the largest is 2^7: FP16's normal numbers end at 2^-14.  Below, each is
    off by 2^-24 / sqrt(12) in the root mean square, where probabilities e^s, s of a variance of one, are 2^-13.2 e
    in theirs: 2^-14, an eighth of 2^-11, which the three roundings' 0.74 (above) leaves room for."""
    c = Cache(lens, H, Hk, D, 16, seed=D + H)
    g = torch.Generator().manual_seed(H)
    total = sum(kv for _, kv in lens)
    q, k, v = (torch.randn(n, h, D, generator=g).half() for n, h in ((c.T, H), (total, Hk), (total, Hk)))
    q[:, :, 0] = 4.0  # a channel that all rows share and only first keys have
    k[:, :, 0] = 0.0
    at = 0
    for _, kv in lens:
        k[at] = 0.0
        k[at, :, 0] = ahead * D ** 0.5 / 4.0
        v[at] *= 2.0 ** -12
        at += kv
    c.fill(k.cuda(), v.cuda())
    out = c.attend(q.cuda(), True)
    capi.sync(stream())
    want = attention64(c, q, quantised(k.float())[0], quantised(v.float())[0], True)
    assert float((out.cpu().double() - want).norm() / want.norm()) <= 2.0 ** -11


def check_attention(c, q, k, v, causal):
    c.fill(k.cuda(), v.cuda())
    out = c.attend(q.cuda(), causal)
    capi.sync(stream())
    (kx, _), (vx, vs) = quantised(k.float()), quantised(v.float())
    want, tol = reference(c, q, kx, vx, vs, causal, c.D ** -0.5)
    bad = (out.cpu().double() - want).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off"
    return out


@pytest.mark.parametrize("seqs,n_max,H,Hk", [(300, 1, 4, 2), (1100, 20, 2, 1)])
def test_many_short_sequences(cuda_dev, seqs, n_max, H, Hk):
    """More sequences than a CTA has threads, some of them without rows or without tokens."""
    g = torch.Generator().manual_seed(seqs)
    lens = []
    for b in range(seqs):
        kv = int(torch.randint(0, 50, (1,), generator=g))
        lens.append((min(kv, 0 if b % 5 == 0 else 1), kv))
    lens[seqs // 2] = (n_max, 90)
    c = Cache(lens, H, Hk, 64, 16, seed=seqs)
    check_attention(c, *held_rows(c, seqs), True)


@pytest.mark.parametrize("D,causal", [(64, True), (128, False)])
def test_many_units_of_one_key_tile(cuda_dev, D, causal):
    """More units a CTA than are published ahead, each of one key tile: half of the operand warps have no tile of
    a unit and meet the next one at once.  More than 32 rows, so that no other kernel takes them."""
    g = torch.Generator().manual_seed(D)
    lens = []
    for b in range(400):
        kv = int(torch.randint(1, 65, (1,), generator=g))
        lens.append((min(kv, 1 + b % 7 * 5), kv))
    c = Cache(lens, 6, 3, D, 16, seed=D)
    q, k, v = held_rows(c, D)
    out = check_attention(c, q, k, v, causal)
    qd = q.cuda()
    for _ in range(20):
        again = c.attend(qd, causal)
        capi.sync(stream())
        assert torch.equal(again, out)


@pytest.mark.parametrize("seed", range(10))
def test_random_batches(cuda_dev, seed):
    """Stretches that begin and end anywhere in sequences of any length."""
    g = torch.Generator().manual_seed(1000 + seed)

    def pick(lo, hi):
        return int(torch.randint(lo, hi + 1, (1,), generator=g))

    Hk, group, D = pick(1, 4), [1, 3, 7, 8][pick(0, 3)], [64, 128][pick(0, 1)]
    n_max = [1, 3, 40, 90][seed % 4]
    lens = []
    for _ in range(pick(1, 14)):
        n = pick(0, n_max)
        lens.append((n, n + pick(0, [40, 700, 3000][pick(0, 2)])))
    lens.append((n_max, n_max + pick(0, 5000)))
    c = Cache(lens, group * Hk, Hk, D, [16, 48, 64][pick(0, 2)], seed=seed)
    check_attention(c, *held_rows(c, seed), seed % 3 != 0)


@pytest.mark.parametrize("n", [1, 50])
@pytest.mark.parametrize("off,pad", [(1, 3), (4, 8)])
def test_attention_strides(cuda_dev, n, off, pad):
    """q and out inside rows of other things, at any alignment of two bytes."""
    c = Cache([(n, 130), (n, 61)], 6, 2, 64, 16, seed=5)
    q, k, v = held_rows(c, 5)
    want = check_attention(c, q, k, v, True)
    ld = 6 * 64 + pad
    qb = torch.full((off + 2 * n * ld,), 3.0, dtype=torch.float16, device="cuda")
    qb[off:].view(2 * n, ld)[:, :384] = q.view(2 * n, 384).cuda()
    ob = torch.full_like(qb, 9.0)
    ws = torch.empty(max(16, c.kv.attention_workspace(c.batch, 6)), dtype=torch.uint8, device="cuda")
    c.kv.attention(c.batch, capi.FP16, qb.data_ptr() + 2 * off, ld, 6, ob.data_ptr() + 2 * off, ld, 0.125, True,
                   ws.data_ptr(), ws.numel(), stream())
    capi.sync(stream())
    got = ob[off:].view(2 * n, ld)
    assert torch.equal(got[:, :384].reshape(want.shape), want)
    assert (got[:, 384:] == 9.0).all() and (ob[:off] == 9.0).all()


@pytest.mark.parametrize("n", [1, 24])
def test_sequences_share_a_prefix(cuda_dev, n):
    """Two sequences whose first pages are the same ones read what each held alone."""
    c = Cache([(n, 100), (n, 80)], 8, 2, 64, 16, seed=6)
    q, k, v = held_rows(c, 6)
    k[100:148], v[100:148] = k[:48], v[:48]
    want = check_attention(c, q, k, v, True)
    c.table[1, :3] = c.table[0, :3]
    out = c.attend(q.cuda(), True)
    capi.sync(stream())
    assert torch.equal(out, want)


@pytest.mark.parametrize("n", [1, 60])
def test_two_calls_at_once(cuda_dev, n):
    """Calls on two streams, each with scratch of its own, give what they give alone."""
    state = []
    for i, kv in enumerate((3000, 700)):
        c = Cache([(n, kv), (1, 200)], 8, 2, 128, 16, seed=i)
        q, k, v = held_rows(c, i)
        c.fill(k.cuda(), v.cuda())
        q = q.cuda()
        want = c.attend(q, True)
        capi.sync(stream())
        ws = torch.empty(max(16, c.kv.attention_workspace(c.batch, 8)), dtype=torch.uint8, device="cuda")
        state.append((c, q, want, ws, [torch.zeros_like(q) for _ in range(6)], torch.cuda.Stream()))
    torch.cuda.synchronize()
    for i in range(6):
        for c, q, _, ws, outs, s in state:
            c.attend(q, True, out=outs[i], st=s.cuda_stream, ws=ws)
    torch.cuda.synchronize()
    capi.sync(stream())
    for _, _, want, _, outs, _ in state:
        for o in outs:
            assert torch.equal(o, want)


@pytest.mark.parametrize("lens", [[(1, 300), (1, 40)], [(150, 300), (20, 40)]])
def test_sharp_and_wide_scores(cuda_dev, lens):
    """Scores of hundreds, one key far ahead of the rest, values of tiny and large scales side by side."""
    c = Cache(lens, 4, 2, 64, 16, seed=5)
    q, k, v = held_rows(c, 6)
    q *= 30
    v[::3] *= 2.0 ** -12
    v[1::7] *= 64
    c.fill(k.cuda(), v.cuda())
    out = c.attend(q.cuda(), True)
    capi.sync(stream())
    (kx, _), (vx, vs) = quantised(k.float()), quantised(v.float())
    want, tol = reference(c, q, kx, vx, vs, True, 64 ** -0.5)
    assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("n,kv", [(3, 40), (140, 150)])
def test_masked_rows_and_stale_pages_do_not_leak(cuda_dev, n, kv):
    """NaN at a position reaches the rows that see it and no other; pages keep what earlier owners left."""
    H, Hk, D = 4, 2, 64
    c = Cache([(n, kv)], H, Hk, D, 16, seed=1)
    q, k, v = held_rows(c, 2)
    # the last page's tail, behind the sequence's end, and one position inside it
    tail = -(-kv // 16) * 16
    if tail > kv:
        t = Cache([(tail, tail)], H, Hk, D, 16, seed=1)
        t.kv = c.kv
        t.table = c.table
        t.ld = c.ld
        full = torch.full((tail, Hk, D), float("nan"), dtype=torch.float16).cuda()
        t.fill(full, full)
    c.fill(k.cuda(), v.cuda())
    clean = c.attend(q.cuda(), True)
    capi.sync(stream())
    assert torch.isfinite(clean).all()
    p = kv - 2
    k2, v2 = k.clone(), v.clone()
    k2[p, 0, 3] = float("nan")
    v2[p, 1, 3] = float("inf")
    c.fill(k2.cuda(), v2.cuda())
    out = c.attend(q.cuda(), True)
    capi.sync(stream())
    sees = torch.arange(kv - n, kv) >= p
    assert torch.equal(out[~sees.cuda()], clean[~sees.cuda()])
    assert torch.isnan(out[sees.cuda()]).all()


def test_pages_beyond_four_gigabytes(cuda_dev):
    lens = [(1, 70), (40, 90)]
    page, Hk, D = 128, 8, 128
    n = (5 << 30) // (page * Hk * (D + 8))
    c = Cache(lens, 16, Hk, D, page, seed=3, pages=n)
    c.table[0, 0], c.table[1, 0] = n - 1, n - 2
    q, k, v = held_rows(c, 3)
    c.fill(k.cuda(), v.cuda())
    out = c.attend(q.cuda(), True)
    capi.sync(stream())
    (kx, _), (vx, vs) = quantised(k.float()), quantised(v.float())
    want, tol = reference(c, q, kx, vx, vs, True, D ** -0.5)
    assert ((out.cpu().double() - want).abs() <= tol).all()
    assert torch.equal(c.read(c.make_batch([70, 90]))[0], kx.half())


@pytest.mark.parametrize("H,n_max", [(8, 1), (8, 40)])
def test_captured_steps_grow(cuda_dev, H, n_max):
    """One captured append + attention, replayed as sequences grow and rows come and go; two graphs with
    scratch of their own at once give what they give alone."""
    Hk, D, cap = 2, 64, 400
    lens = [(n_max, cap), (n_max, cap)]
    g = torch.Generator().manual_seed(1)
    caches = [Cache(lens, H, Hk, D, 16, 10000.0, seed=i) for i in range(2)]
    total = 2 * n_max
    state = []
    for c in caches:
        q, k, v = (rows(g, total, h, D).cuda() for h in (H, Hk, Hk))
        b = c.make_batch([n_max, n_max], held=[n_max, n_max])
        ws = torch.full((max(16, c.kv.attention_workspace(b, H)),), 255, dtype=torch.uint8, device="cuda")
        qo, out = torch.zeros_like(q), torch.zeros_like(q)
        graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            st = torch.cuda.current_stream().cuda_stream
            c.append(b, k, v, q, qo, st)
            c.attend(qo, True, batch=b, out=out, st=st, ws=ws)
        state.append((c, b, q, k, v, qo, out, graph, s))
    for step in range(4):
        want = []
        for c, b, q, k, v, qo, out, graph, s in state:
            new = [n_max, 0] if step == 2 else [1, n_max]
            held = [n_max + 97 * step, n_max + 31 * step]
            b.keep[0].copy_(torch.tensor([0, new[0], new[0] + new[1]], dtype=torch.int32))
            b.keep[1].copy_(torch.tensor(held, dtype=torch.int32))
            for t in (q, k, v):
                t.copy_(rows(g, *t.shape).cuda())
            out.fill_(9.0)
            c.append(b, k, v, q, qo)
            ref = torch.full_like(q, 9.0)
            c.attend(qo, True, batch=b, out=ref)
            capi.sync(stream())
            want.append(ref)
        torch.cuda.synchronize()
        for *_, graph, s in state:
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for w, (c, b, q, k, v, qo, out, graph, s) in zip(want, state):
            assert torch.equal(out, w)
    capi.sync(stream())


def test_decode_step_in_four_bits(cuda_dev):
    """q, k, v product -> append with rotation -> attention -> output product, as a decode step runs them, for
    three steps behind a prompt, against the same in 64 bits on the held values."""
    hidden, H, Hk, D, theta, B = 256, 4, 2, 64, 10000.0, 3
    prompt, steps = [37, 5, 120], 3
    c = Cache([(1, p + steps) for p in prompt], H, Hk, D, 16, theta, seed=7)
    g = torch.Generator().manual_seed(8)
    wide = (H + 2 * Hk) * D
    src = [(torch.randn(n, k, generator=g) / k ** 0.5).half().cuda() for n, k in ((wide, hidden), (hidden, H * D))]
    w1, w2 = (capi.WeightQ4(t.data_ptr(), capi.FP16, True, t.shape[0], t.shape[1], 64, False, stream()) for t in src)
    vals = []
    for w, t in zip((w1, w2), src):
        r = torch.empty_like(t)
        w.read(r.data_ptr(), stream=stream())
        capi.sync(stream())
        vals.append(r.double().cpu())
    kp, vp = rows(g, sum(prompt), Hk, D), rows(g, sum(prompt), Hk, D)
    c.append(c.make_batch(prompt, held=prompt), kp.cuda(), vp.cuda())
    kr, vr = [t.double() for t in c.read(c.make_batch(prompt, held=prompt))]
    x = torch.randn(B, hidden, generator=g).half().cuda()
    hist = [(kr[sum(prompt[:b]):sum(prompt[:b + 1])], vr[sum(prompt[:b]):sum(prompt[:b + 1])]) for b in range(B)]
    for step in range(steps):
        held = [p + step + 1 for p in prompt]
        b = c.make_batch([1] * B, held=held)
        qkv = torch.empty(B, wide, dtype=torch.float16, device="cuda")
        attn, y = torch.empty(B, H * D, dtype=torch.float16, device="cuda"), x.clone()
        capi.gemv_q4(w1, x.data_ptr(), hidden, qkv.data_ptr(), wide, B, stream=stream())
        p = qkv.data_ptr()
        c.kv.append(b, capi.FP16, p, wide, H, p, wide, p + 2 * H * D, wide, p + 2 * (H + Hk) * D, wide, stream())
        n = c.kv.attention_workspace(b, H)
        ws = torch.empty(max(16, n), dtype=torch.uint8, device="cuda")
        c.kv.attention(b, capi.FP16, p, wide, H, attn.data_ptr(), H * D, D ** -0.5, True, ws.data_ptr(), ws.numel(),
                       stream())
        capi.gemv_q4(w2, attn.data_ptr(), H * D, y.data_ptr(), hidden, B, res_ptr=y.data_ptr(), ldr=hidden,
                     stream=stream())
        capi.sync(stream())
        kn, vn = [t.double() for t in c.read(b)]
        want = x.cpu().double() @ vals[0].t()
        want = want.view(B, -1, D)
        pos = torch.tensor(held) - 1
        q = rotated(want[:, :H], pos, theta)
        o = torch.empty(B, H, D, dtype=torch.float64)
        for i in range(B):
            hist[i] = (torch.cat((hist[i][0], kn[i:i + 1])), torch.cat((hist[i][1], vn[i:i + 1])))
            kk, vv = hist[i]
            s = torch.einsum("hgd,thd->hgt", q[i].view(Hk, -1, D), kk) * D ** -0.5
            o[i] = torch.einsum("hgt,thd->hgd", s.softmax(-1), vv).reshape(H, D)
        want = x.cpu().double() + o.view(B, -1) @ vals[1].t()
        got = y.cpu().double()
        # five FP16 roundings on the way (q k v, rotated q, values read here, attention, output), each 2^-11
        assert float((got - want).norm() / want.norm()) <= 5 * 2.0 ** -11
        x = y


def test_bad_pages_and_lengths_are_reported(cuda_dev):
    H, Hk, D = 2, 1, 64
    c = Cache([(1, 20), (1, 30)], H, Hk, D, 16, seed=1)
    q, k, v = held_rows(c, 1)
    c.fill(k.cuda(), v.cuda())
    good = c.attend(q.cuda(), True)
    capi.sync(stream())
    keep = c.table.clone()
    for bad in (-1, 10 ** 6):
        c.table[0, 1] = bad
        out = c.attend(q.cuda(), True)
        with pytest.raises(capi.MrtError) as e:
            capi.sync(stream())
        assert e.value.code == 1
        assert torch.equal(out[1], good[1])
        last = [19, 49]  # what the two positions hold already: the good sequence's row is stored again
        c.append(c.batch, k[last].cuda(), v[last].cuda())
        with pytest.raises(capi.MrtError):
            capi.sync(stream())
        c.table.copy_(keep)
    for held, new in (([200, 30], [1, 1]), ([20, -3], [1, 1]), ([20, 30], [2, 1])):
        b = c.make_batch(new, tokens=3, held=held, max_q=1, max_kv=32)
        qq = torch.zeros(3, H, D, dtype=torch.float16, device="cuda")
        c.attend(qq, True, batch=b)
        with pytest.raises(capi.MrtError):
            capi.sync(stream())
    again = c.attend(q.cuda(), True)
    capi.sync(stream())
    assert torch.equal(again, good)


# q_start and kv_len of two sequences, of calls with 4 rows, at most 4 a sequence and 32 tokens held; the rows that are good
BAD_LENGTHS = [([0, 4, 8], [20, 30], [0, 1, 2, 3]), ([0, 2, 5], [20, 30], [0, 1]), ([4, 4, 5], [20, 30], []),
               ([0, 3, 2], [20, 30], [0, 1, 2]), ([0, 4, 4], [20, 33], [0, 1, 2, 3]), ([0, 0, 4], [-1, 30], [0, 1, 2, 3]),
               ([0, 1, 4], [33, 30], [1, 2, 3]), ([-1, 2, 4], [20, 30], [2, 3])]


@pytest.mark.parametrize("case", range(len(BAD_LENGTHS)))
@pytest.mark.parametrize("heads", [2, 16])
def test_every_call_reports_bad_lengths(cuda_dev, case, heads):
    """Append, read and attention (of few rows and of many) leave a bad sequence's rows as they were, serve the
    other, and say so: a sequence behind the call's rows, one without rows and one that ends before it begins too."""
    start, held, good = BAD_LENGTHS[case]
    D = 64
    c = Cache([(4, 32), (4, 32)], heads, 1, D, 16, 10000.0, seed=case)
    g = torch.Generator().manual_seed(case)
    k, v = rows(g, 64, 1, D), rows(g, 64, 1, D)
    c.fill(k.cuda(), v.cuda())
    b = c.make_batch([0, 0], tokens=4, max_q=4, max_kv=32)
    b.keep[0].copy_(torch.tensor(start, dtype=torch.int32))
    b.keep[1].copy_(torch.tensor(held, dtype=torch.int32))
    q = rows(g, 4, heads, D).cuda()
    qo, kn, vn = torch.full_like(q, 9.0), rows(g, 4, 1, D).cuda(), rows(g, 4, 1, D).cuda()
    rest = [i for i in range(4) if i not in good]

    def reported():
        with pytest.raises(capi.MrtError) as e:
            capi.sync(stream())
        assert e.value.code == 1

    c.append(b, kn, vn, q, qo)
    reported()
    assert (qo[rest] == 9.0).all() and all((qo[i] != 9.0).any() for i in good)
    kr, vr = (torch.full((4, 1, D), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    c.kv.read(b, capi.FP16, kr.data_ptr(), D, vr.data_ptr(), D, stream())
    reported()
    assert (vr[rest] == 9.0).all()
    assert torch.equal(vr[good].cpu(), quantised(vn[good].cpu().float())[0].half())
    out = c.attend(q, True, batch=b)
    reported()
    assert (out[rest] == 9.0).all() and all((out[i] != 9.0).any() for i in good)


@pytest.mark.parametrize("n,kv,H", [(3, 33, 4), (3, 33, 8), (40, 49, 4)])
def test_a_bad_page_spoils_no_row_that_does_not_need_it(cuda_dev, n, kv, H):
    """The newest token's page is none of the cache: earlier rows do not see it."""
    c = Cache([(n, kv)], H, 2, 64, 16, seed=4)
    q, k, v = held_rows(c, 4)
    good = check_attention(c, q, k, v, True)
    c.table[0, kv // 16] = 10 ** 6
    out = c.attend(q.cuda(), True)
    with pytest.raises(capi.MrtError):
        capi.sync(stream())
    sees = torch.arange(kv - n, kv) >= kv // 16 * 16
    assert torch.equal(out[~sees.cuda()], good[~sees.cuda()])


def test_refusals(cuda_dev):
    c = Cache([(1, 20)], 4, 2, 64, 16)
    t = torch.zeros(4096, dtype=torch.float16, device="cuda")
    p, L = t.data_ptr(), capi.lib()
    import ctypes as C

    def batch(**kw):
        a = dict(seqs=1, tokens=1, max_q_len=1, max_kv_len=20, q_start_dev=c.batch.q_start_dev,
                 kv_len_dev=c.batch.kv_len_dev, table_dev=c.table.data_ptr(), ld_table=c.ld)
        a.update(kw)
        return capi.KvBatch(**a)

    def append(b=None, dt=0, q=p, ldq=256, heads=4, qo=p, ldqo=256, k=p, ldk=128, v=p, ldv=128):
        return L.mrt_kv_q4_append(c.kv.h, C.byref(b or batch()), dt, q, ldq, heads, qo, ldqo, k, ldk, v, ldv, stream())

    def attend(b=None, dt=0, q=p, ldq=256, heads=4, o=p, ldo=256, ws=None, n=None):
        ws = c_ws.data_ptr() if ws is None else ws
        return L.mrt_kv_q4_attention(c.kv.h, C.byref(b or batch()), dt, q, ldq, heads, o, ldo, 0.1, 1, ws or None,
                                     c_ws.numel() if n is None else n, stream())

    c_ws = torch.empty(max(16, c.kv.attention_workspace(batch(), 4)), dtype=torch.uint8, device="cuda")
    for f in (append, attend):
        assert f() == 0 and f(batch(seqs=0)) == 0 and f(batch(tokens=0)) == 0
        for kw in (dict(seqs=-1), dict(tokens=-1), dict(max_q_len=-1), dict(max_kv_len=-1), dict(seqs=65536),
                   dict(tokens=1 << 31), dict(max_kv_len=c.ld * 16 + 1)):
            assert f(batch(**kw)) == 2, kw
        for kw in (dict(q_start_dev=None), dict(kv_len_dev=None), dict(table_dev=None)):
            assert f(batch(**kw)) == 1, kw
        assert f(dt=2) == 3 and f(q=None) == 1 and f(ldq=255) == 2
    assert append(k=None) == 1 and append(v=None) == 1 and append(qo=None) == 1 and append(heads=-1) == 2
    assert append(ldk=127) == 2 and append(ldv=127) == 2 and append(ldqo=255) == 2
    assert append(q=None, qo=None, heads=0) == 0
    assert attend(o=None) == 1 and attend(ldo=255) == 2 and attend(heads=3) == 2 and attend(heads=0) == 2
    assert L.mrt_kv_q4_read(c.kv.h, C.byref(batch()), 2, p, 128, p, 128, stream()) == 3
    assert L.mrt_kv_q4_read(c.kv.h, C.byref(batch()), 0, p, 127, p, 128, stream()) == 2
    assert L.mrt_kv_q4_read(c.kv.h, C.byref(batch()), 0, None, 0, None, 0, stream()) == 0
    capi.sync(stream())
