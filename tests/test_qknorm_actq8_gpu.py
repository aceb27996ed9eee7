"""The norm of queries and keys with the rotation, and the 8-bit activation checkpoints, against their formulas in 64 bits.

Tolerances are bounds by arithmetic.  u = 2^-24 is half a step of fp32, half(T) half a step of the output's type relative to the
value (2^-8 for bf16, 2^-24 for fp32).  A sum of n terms in fp32 is off by at most n u times the sum of their magnitudes.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [0, 1]


@pytest.fixture(scope='module')
def K():
    from s4former_amd import kernels
    return kernels


def tdt(code):
    return torch.bfloat16 if code == 1 else torch.float32


def half(code):
    return torch.finfo(tdt(code)).eps / 2


def rnd(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


def within(got, ref, tol, what):
    got, ref = got.detach().cpu().double(), ref.double()
    assert got.shape == ref.shape, f'{what}: {tuple(got.shape)} vs {tuple(ref.shape)}'
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), f'{what}: {int(bad.sum())} of {bad.numel()} outside, worst excess {((got - ref).abs() - tol).max():.3e}'


def sliced(t, pad, code):
    """the matrix as a column slice of a wider device buffer (pad extra columns on both sides, filled with NaN)"""
    t = t.to(tdt(code))
    if pad == 0:
        return t.contiguous().cuda()
    buf = torch.full((t.shape[0], t.shape[1] + 2 * pad), float('nan'), dtype=t.dtype, device='cuda')
    buf[:, pad:pad + t.shape[1]] = t.cuda()
    return buf[:, pad:pad + t.shape[1]]


# ------------------------------------------------------------------------------------------------------------- plain forms, 64 bits
def q8_plain(x):
    """codes (int64) and scales (2^k, 64 bits) of a [rows, C] tensor; NaN scales for groups that are not finite"""
    g = x.double().reshape(x.shape[0], -1, 32)
    amax = g.abs().amax(-1)
    finite = torch.isfinite(g).all(-1)
    e = torch.full_like(amax, -126.0)
    for k in range(-126, 121):                               # the least power of two with round(amax / s) <= 127, 2^121 at most
        s = 2.0 ** k
        e = torch.where(torch.round(torch.where(finite, amax, torch.zeros_like(amax)) / s) > 127, torch.full_like(e, k + 1.0), e)
    s = torch.exp2(e)
    codes = torch.where(finite[..., None], torch.round(g / s[..., None]).clamp(-127, 127), torch.zeros_like(g))
    s = torch.where(finite, s, torch.full_like(s, float('nan')))
    return codes.reshape(x.shape), s


def q8_restore(codes, s):
    return (codes.reshape(codes.shape[0], -1, 32) * s[..., None]).reshape(codes.shape)


def tables(period, seed=0, per_row=False):
    pos = torch.arange(period, dtype=torch.float64)[:, None] + 37 * seed
    ang = pos * 100.0 ** (-torch.arange(32, dtype=torch.float64) / 32)
    return ang.cos().float(), ang.sin().float()


def turn(v, cos, sin, sign):
    """v [rows, H, 64], tables [period, 32]"""
    n = v.shape[0] // cos.shape[0]
    c, s = cos.double().repeat(n, 1)[:, None], sign * sin.double().repeat(n, 1)[:, None]
    lo, hi = v[..., :32], v[..., 32:]
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1)


def qk_plain(x, Hq, Hk, gq, gk, cos, sin, eps):
    """(y, magnitudes that the rounding errors of y are relative to)"""
    v = x.double().reshape(x.shape[0], Hq + Hk, 64)
    if gq is not None:
        g = torch.cat([gq.double().expand(Hq, 64), gk.double().expand(Hk, 64)])
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * g
    mag = v.abs()
    if cos is not None:
        mag = (mag[..., :32] + mag[..., 32:]).repeat(1, 1, 2)
        v = turn(v, cos, sin, 1.0)
    return v.reshape(x.shape), mag.reshape(x.shape)


def qk_plain_bwd(dy, x, Hq, Hk, gq, gk, cos, sin, eps):
    """(dx, magnitude, dgq, magnitude, dgk, magnitude)"""
    H = Hq + Hk
    dz = dy.double().reshape(-1, H, 64)
    mag = dz.abs()
    if cos is not None:
        mag = (mag[..., :32] + mag[..., 32:]).repeat(1, 1, 2)
        dz = turn(dz, cos, sin, -1.0)
    if gq is None:
        return dz.reshape(dy.shape), mag.reshape(dy.shape), None, None, None, None
    x = x.double().reshape(-1, H, 64)
    g = torch.cat([gq.double().expand(Hq, 64), gk.double().expand(Hk, 64)])
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    u = x * r
    dx = r * (dz * g - u * (dz * g * u).mean(-1, keepdim=True))
    dmag = r * (mag * g.abs() + u.abs() * (mag * (g * u).abs()).mean(-1, keepdim=True))
    dg, gm = (dz * u).sum(0), (mag * u.abs()).sum(0)
    return dx.reshape(dy.shape), dmag.reshape(dy.shape), dg[:Hq].sum(0), gm[:Hq].sum(0), dg[Hq:].sum(0), gm[Hq:].sum(0)


# rounding steps of the kernels (see the bounds above): forward - 64 squares and eps through a root (half of 66), root 2, two
# products, three of the rotation: below 48; backward - the same for u, 64 terms of the mean and its products: below 160
FWD_STEPS, BWD_STEPS = 48, 160


def gain_steps(items):
    # u and dz (60), a lane's own items in sequence, at most 64 + 16 partial sums in the join and 8 in the block
    return 60 + items / 32768 + 2 + 64 + 16 + 8


QK_CASES = [
    # B, N, Hq, Hk, norm, rope, per-image positions, pad
    (1, 1, 1, 1, True, True, False, 0),
    (1, 1, 4, 1, True, False, False, 64),
    (2, 17, 4, 4, True, True, False, 0),
    (3, 5, 3, 2, True, True, True, 32),
    (2, 33, 12, 12, False, True, True, 8),
    (1, 197, 16, 2, True, False, False, 0),
    (5, 129, 6, 6, True, True, True, 128),
]


def qk_inputs(case, code, seed=0):
    B, N, Hq, Hk, norm, rope, own, pad = case
    rows, C = B * N, (Hq + Hk) * 64
    x = (rnd(rows, C, seed=seed + 1) * torch.exp(rnd(1, C, seed=seed + 2))).to(tdt(code)).float()
    x[0, :64] = 0                                            # a head of zeros
    dy = rnd(rows, C, seed=seed + 3, scale=0.1).to(tdt(code)).float()
    gq, gk = (1 + 0.3 * rnd(64, seed=seed + 4), 1 + 0.3 * rnd(64, seed=seed + 5)) if norm else (None, None)
    if norm:
        gq[3] = 0                                            # a gain of zero
    cos, sin = tables(rows if own else N, seed) if rope else (None, None)
    return x, dy, gq, gk, cos, sin


def cu(t):
    return None if t is None else t.cuda()


@pytest.mark.parametrize('code', DTYPES)
@pytest.mark.parametrize('case', QK_CASES)
def test_qk_forward(K, code, case):
    B, N, Hq, Hk, norm, rope, own, pad = case
    x, _, gq, gk, cos, sin = qk_inputs(case, code)
    C, eps = (Hq + Hk) * 64, 1e-6
    xs = sliced(x, pad, code)
    y = sliced(torch.zeros_like(x), 2 * pad, code)
    whole = y if pad == 0 else y._base
    before = whole.clone()
    par = dict(gq=cu(gq), gk=cu(gk), cos=cu(cos), sin=cu(sin), eps=eps)
    K.qk_norm_rope_fwd(xs, y, Hq, Hk, code, **par)
    ref, mag = qk_plain(x, Hq, Hk, gq, gk, cos, sin, eps)
    within(y, ref, half(code) * ref.abs() + FWD_STEPS * U * mag * (1 + half(code)), 'y')
    if pad:                                                  # the columns beside the slice are left as they were
        keep = torch.ones(whole.shape[1], dtype=torch.bool)
        keep[2 * pad:2 * pad + C] = False
        assert torch.equal(whole[:, keep].isnan(), before[:, keep].isnan()) and bool(whole[:, keep].isnan().all())
    inplace = sliced(x, pad, code)
    K.qk_norm_rope_fwd(inplace, inplace, Hq, Hk, code, **par)
    assert torch.equal(inplace, y)


@pytest.mark.parametrize('code', DTYPES)
@pytest.mark.parametrize('from_packed', [False, True])
@pytest.mark.parametrize('case', QK_CASES)
def test_qk_backward(K, code, from_packed, case):
    B, N, Hq, Hk, norm, rope, own, pad = case
    if from_packed and not norm:
        pytest.skip('the rotation alone keeps nothing')
    x, dy, gq, gk, cos, sin = qk_inputs(case, code, seed=10)
    rows, C, eps = B * N, (Hq + Hk) * 64, 1e-6
    par = dict(gq=cu(gq), gk=cu(gk), cos=cu(cos), sin=cu(sin), eps=eps)
    xs, kept = sliced(x, pad, code), x.double()
    kw = dict(x=xs) if norm else {}
    if from_packed:
        codes = torch.empty(rows, C, device='cuda', dtype=torch.int8)
        scales = torch.empty(rows, C // 32, device='cuda', dtype=torch.uint8)
        y0, y1 = torch.empty(rows, C, device='cuda', dtype=tdt(code)), torch.empty(rows, C, device='cuda', dtype=tdt(code))
        K.qk_norm_rope_fwd(xs, y0, Hq, Hk, code, **par)
        K.qk_norm_rope_fwd(xs, y1, Hq, Hk, code, packed=(codes, scales), **par)
        assert torch.equal(y0, y1)
        c2, s2 = torch.empty_like(codes), torch.empty_like(scales)
        K.act_pack(xs, c2, s2, code)                         # the checkpoint is the one of act_pack
        assert torch.equal(codes, c2) and torch.equal(scales, s2)
        cr, sr = q8_plain(x)
        assert torch.equal(codes.cpu().double(), cr)
        kept = q8_restore(cr, sr)
        kw = dict(packed=(codes, scales))
    dys = sliced(dy, pad, code)
    base = [rnd(64, seed=20), rnd(64, seed=21)]
    dg = [b.cuda() for b in base]
    ws = torch.full((max(1, K.qk_norm_rope_ws_bytes(rows, Hq, Hk) // 4),), float('nan'), device='cuda')
    dx = torch.empty(rows, C, device='cuda', dtype=tdt(code))
    grads = dict(dgq=dg[0], dgk=dg[1], ws=ws) if norm else {}
    K.qk_norm_rope_bwd(dys, dx, Hq, Hk, code, **kw, **par, **grads)
    rdx, mdx, rq, mq, rk, mk = qk_plain_bwd(dy, kept, Hq, Hk, gq, gk, cos, sin, eps)
    within(dx, rdx, half(code) * rdx.abs() + BWD_STEPS * U * mdx * (1 + half(code)), 'dx')
    if norm:
        for got, b, ref, mag, heads, what in ((dg[0], base[0], rq, mq, Hq, 'dgq'), (dg[1], base[1], rk, mk, Hk, 'dgk')):
            within(got, b.double() + ref, gain_steps(rows * heads) * U * mag + U * (b.abs() + ref.abs()) * 2, what)
        fresh = [torch.full((64,), float('nan'), device='cuda') for _ in range(2)]
        again = sliced(dy, pad, code)
        K.qk_norm_rope_bwd(again, again, Hq, Hk, code, dgq=fresh[0], dgk=fresh[1], ws=ws, accumulate=False, **kw, **par)   # in place
        assert torch.equal(again, dx)
        within(fresh[0], rq, gain_steps(rows * Hq) * U * mq + U * rq.abs(), 'dgq written')


@pytest.mark.parametrize('norm,rope', [(True, True), (True, False), (False, True)])
def test_qk_backward_against_differences(K, norm, rope):
    """fp32 gradients against central differences of the 64-bit forward along random directions"""
    case = (2, 9, 2, 1, norm, rope, False, 0)
    x, dy, gq, gk, cos, sin = qk_inputs(case, 0, seed=30)
    x[0, :64] = rnd(64, seed=31)                             # (a head of zeros has curvature 1 / eps)
    Hq, Hk, eps = 2, 1, 1e-6
    dx = torch.empty_like(x).cuda()
    par = dict(gq=cu(gq), gk=cu(gk), cos=cu(cos), sin=cu(sin), eps=eps)
    dg = [torch.zeros(64, device='cuda') for _ in range(2)]
    ws = torch.empty(K.qk_norm_rope_ws_bytes(18, Hq, Hk), device='cuda', dtype=torch.uint8)
    kw = dict(x=x.cuda(), dgq=dg[0], dgk=dg[1], ws=ws) if norm else {}
    K.qk_norm_rope_bwd(dy.cuda(), dx, Hq, Hk, 0, **kw, **par)

    def f(x_, gq_, gk_):
        return (qk_plain(x_, Hq, Hk, gq_, gk_, cos, sin, eps)[0] * dy.double()).sum()
    h = 1e-5
    d = rnd(*x.shape, seed=33).double()
    num = (f(x.double() + h * d, gq, gk) - f(x.double() - h * d, gq, gk)) / (2 * h)
    ana = (dx.cpu().double() * d).sum()
    # central differences are off by h^2 f''' / 6 (about 1e-10 of the terms), the kernel by fp32 rounding of each term
    tol = (BWD_STEPS * U * 4 + 1e-7) * (dx.cpu().double() * d).abs().sum()
    assert abs(num - ana) <= tol, (num, ana, tol)
    if norm:
        d = rnd(64, seed=34).double()
        num = (f(x, gq.double() + h * d, gk) - f(x, gq.double() - h * d, gk)) / (2 * h)
        ana = (dg[0].cpu().double() * d).sum()
        assert abs(num - ana) <= 1e-5 * (dg[0].cpu().double() * d).abs().sum(), (num, ana)


# B, N, Hq, Hk: so many heads that the backward's grid is capped, a lane takes several of them (a ragged number) and the join of the gains
# more than one turn
MANY_CASES = [(8, 1025, 12, 12), (3, 2305, 16, 4)]


def kind_blocks(rows, heads, all_heads, packed, code):
    """(blocks of the backward for the heads of one kind, heads that a block takes at a time)"""
    per, most = 64 if packed and code == 1 else 32, 1024 if packed else 768
    return min(-(-rows * heads // per), max(1, most * heads // all_heads)), per


def many_gain_steps(rows, heads, all_heads, packed, code):
    blocks, per = kind_blocks(rows, heads, all_heads, packed, code)
    lane, turns = -(-rows * heads // (blocks * per)), -(-blocks // 256)
    # u and dz (60); a lane's own heads; the lanes of a wave (at most 4 exchanges) and its 4 waves; the join: a thread's turns, 6 exchanges, 4 waves
    return 60 + lane + 4 + 4 + turns + 6 + 4


@pytest.mark.parametrize('code', DTYPES)
@pytest.mark.parametrize('packed', [False, True])
@pytest.mark.parametrize('case', MANY_CASES)
def test_many_heads_backward(K, code, packed, case):
    """dx and the gains' gradients at sizes of a real batch, each kind of head by its own number of blocks"""
    B, N, Hq, Hk = case
    rows, H, C, eps = B * N, Hq + Hk, (Hq + Hk) * 64, 1e-6
    blocks = [kind_blocks(rows, h, H, packed, code) for h in (Hq, Hk)]
    assert max(b for b, _ in blocks) > 256 and all(rows * h > b * per for (b, per), h in zip(blocks, (Hq, Hk)))
    gen = torch.Generator(device='cuda').manual_seed(rows)
    x = (torch.randn(rows, C, device='cuda', generator=gen) * torch.exp(0.3 * torch.randn(1, C, device='cuda', generator=gen))).to(tdt(code))
    dy = (0.1 * torch.randn(rows, C, device='cuda', generator=gen)).to(tdt(code))
    gq, gk = [1 + 0.3 * torch.randn(64, device='cuda', generator=gen) for _ in range(2)]
    cos, sin = [t.cuda() for t in tables(N)]
    kept, kw = x.double(), dict(x=x)
    if packed:
        codes, scales = torch.empty(rows, C, device='cuda', dtype=torch.int8), torch.empty(rows, C // 32, device='cuda', dtype=torch.uint8)
        K.act_pack(x, codes, scales, code)
        kept, kw = q8_restore(codes.double(), torch.exp2(scales.double() - 127)), dict(packed=(codes, scales))
    dx = torch.empty_like(x)
    dg = [torch.full((64,), float('nan'), device='cuda') for _ in range(2)]
    ws = torch.full((K.qk_norm_rope_ws_bytes(rows, Hq, Hk) // 4,), float('nan'), device='cuda')
    par = dict(gq=gq, gk=gk, cos=cos, sin=sin, eps=eps, ws=ws)
    K.qk_norm_rope_bwd(dy, dx, Hq, Hk, code, dgq=dg[0], dgk=dg[1], accumulate=False, **kw, **par)
    rdx, mdx, rq, mq, rk, mk = qk_plain_bwd(dy, kept, Hq, Hk, gq, gk, cos, sin, eps)
    within(dx, rdx.cpu(), (half(code) * rdx.abs() + BWD_STEPS * U * mdx * (1 + half(code))).cpu(), 'dx')
    steps = [many_gain_steps(rows, h, H, packed, code) for h in (Hq, Hk)]
    within(dg[0], rq.cpu(), (steps[0] * U * mq).cpu(), 'dgq')
    within(dg[1], rk.cpu(), (steps[1] * U * mk).cpu(), 'dgk')
    before = [g.clone() for g in dg]
    K.qk_norm_rope_bwd(dy, dx, Hq, Hk, code, dgq=dg[0], dgk=dg[1], **kw, **par)                       # added: one more rounding
    for g, b in zip(dg, before):
        assert torch.equal(g, b + b)


@pytest.mark.parametrize('code', DTYPES)
@pytest.mark.parametrize('packed', [False, True])
@pytest.mark.parametrize('case', MANY_CASES)
def test_gain_sums_lose_nothing(K, code, packed, case):
    """x of +1 and -1 (mean 1, an eps that vanishes beside it: u = x), whole dy and quarter turns: every operation is exact and every sum a whole
    number below 2^24, so one head that is left out or taken twice shows"""
    B, N, Hq, Hk = case
    rows, H, C = B * N, Hq + Hk, (Hq + Hk) * 64
    gen = torch.Generator(device='cuda').manual_seed(rows + 1)
    x = (torch.randint(0, 2, (rows, C), device='cuda', generator=gen) * 2 - 1).to(tdt(code))
    dy = torch.randint(-3, 4, (rows, C), device='cuda', generator=gen).to(tdt(code))
    quarter = torch.randint(0, 4, (N, 32), device='cuda', generator=gen)
    cos, sin = [torch.tensor(v, device='cuda')[quarter] for v in ([1.0, 0.0, -1.0, 0.0], [0.0, 1.0, 0.0, -1.0])]
    gain = torch.ones(64, device='cuda')
    kw = dict(x=x)
    if packed:
        kw = dict(packed=(torch.empty(rows, C, device='cuda', dtype=torch.int8), torch.empty(rows, C // 32, device='cuda', dtype=torch.uint8)))
        K.act_pack(x, *kw['packed'], code)
    dx = torch.empty_like(x)
    dg = [torch.empty(64, device='cuda') for _ in range(2)]
    ws = torch.empty(K.qk_norm_rope_ws_bytes(rows, Hq, Hk), device='cuda', dtype=torch.uint8)
    K.qk_norm_rope_bwd(dy, dx, Hq, Hk, code, gq=gain, gk=gain, cos=cos, sin=sin, eps=2.0 ** -126, dgq=dg[0], dgk=dg[1], ws=ws, accumulate=False, **kw)
    each = (turn(dy.double().reshape(rows, H, 64), cos, sin, -1.0) * x.double().reshape(rows, H, 64)).sum(0)
    assert torch.equal(dg[0].double(), each[:Hq].sum(0)) and torch.equal(dg[1].double(), each[Hq:].sum(0))


# ------------------------------------------------------------------------------------------------------------- checkpoints
PACK_CASES = [(1, 32, 0), (1, 352, 8), (3, 64, 0), (65, 768, 0), (7, 1056, 8), (130, 256, 640), (1025, 96, 32)]


@pytest.mark.parametrize('code', DTYPES)
@pytest.mark.parametrize('rows,C,pad', PACK_CASES)
def test_pack_unpack(K, code, rows, C, pad):
    x = rnd(rows, C, seed=rows + C) * torch.exp(3 * rnd(rows, C // 32, seed=2)).repeat_interleave(32, 1)
    x = x.to(tdt(code)).float()
    xs = sliced(x, pad, code)
    codes = torch.full((rows, C), 77, device='cuda', dtype=torch.int8)
    scales = torch.full((rows, C // 32), 77, device='cuda', dtype=torch.uint8)
    K.act_pack(xs, codes, scales, code)
    cr, sr = q8_plain(x)
    assert torch.equal(codes.cpu().double(), cr)
    assert torch.equal(torch.exp2(scales.cpu().double() - 127), sr)
    y = sliced(torch.zeros_like(x), pad, code)
    K.act_unpack(codes, scales, y, code)
    assert torch.equal(y.cpu().double(), q8_restore(cr, sr))                      # exact, in either type
    amax = x.double().reshape(rows, -1, 32).abs().amax(-1).repeat_interleave(32, 1)
    assert ((y.cpu().double() - x.double()).abs() <= amax / 63.75 / 2).all()
    if pad:
        assert bool(y._base[:, :pad].isnan().all()) and bool(y._base[:, pad + C:].isnan().all())


@pytest.mark.parametrize('code', DTYPES)
def test_pack_values_at_the_edges(K, code):
    """rounding ties, the border of a scale, the smallest and largest magnitudes, infinities and NaN"""
    t = tdt(code)
    rows = [torch.zeros(32)]
    for top in (127.0, 127.5, 128.0, 63.5, 64.0, 127.25):
        r = torch.arange(32, dtype=torch.float32) - 15.5                          # halves: ties to even
        r[0] = top
        rows.append(r)
        rows.append(-r)
    rows.append(torch.full((32,), torch.finfo(t).max))
    rows.append(torch.full((32,), -torch.finfo(t).tiny))
    rows.append(torch.full((32,), 2.0 ** -130))                                   # below the normal range
    rows.append(2.0 ** -120 * (torch.arange(32) - 16.0))
    n = len(rows)
    for bad in (float('inf'), float('-inf'), float('nan')):
        r = rnd(32, seed=5)
        r[7] = bad
        rows.append(r)
    x = torch.stack(rows).to(t).float()
    codes = torch.empty(len(rows), 32, device='cuda', dtype=torch.int8)
    scales = torch.empty(len(rows), 1, device='cuda', dtype=torch.uint8)
    y = torch.empty(len(rows), 32, device='cuda', dtype=t)
    K.act_pack(x.to(t).cuda(), codes, scales, code)
    K.act_unpack(codes, scales, y, code)
    cr, sr = q8_plain(x)
    assert torch.equal(codes.cpu().double(), cr)
    assert torch.equal(scales.cpu()[:n].double().sub(127).exp2(), sr[:n]) and bool((scales.cpu()[n:] == 255).all())
    assert torch.equal(y.cpu()[:n].double(), q8_restore(cr[:n], sr[:n])) and bool(y[n:].isnan().all())
    amax = x[:n].double().abs().amax(1, keepdim=True)
    assert ((y.cpu()[:n].double() - x[:n].double()).abs() <= torch.clamp(amax / 127.5, min=2.0 ** -127)).all()


def test_pack_leaves_other_rows(K):
    """rows behind the last one, and a buffer that is longer than needed, stay as they were"""
    x = rnd(5, 64, seed=1).cuda()
    codes = torch.full((9, 64), 5, device='cuda', dtype=torch.int8)
    scales = torch.full((9, 2), 5, device='cuda', dtype=torch.uint8)
    K.act_pack(x, codes[:5], scales[:5], 0)
    assert bool((codes[5:] == 5).all()) and bool((scales[5:] == 5).all())
    y = torch.full((9, 64), 5.0, device='cuda')
    K.act_unpack(codes[:5], scales[:5], y[:5], 0)
    assert bool((y[5:] == 5).all())


# ------------------------------------------------------------------------------------------------------------- weight gradients
WG_CASES = [
    # rows, [(M, N), ...], pad
    (1, [(8, 32)], 0),
    (31, [(24, 96)], 8),
    (33, [(136, 160)], 0),
    (64, [(128, 128)], 0),
    (257, [(264, 288)], 16),
    (700, [(256, 256), (8, 512), (384, 32)], 0),
    (1025, [(256, 768), (768, 256), (256, 256), (768, 256)], 8),
    (4100, [(512, 512)], 0),
]


def packed_inputs(rows, shapes, code, seed, pad=0):
    out = []
    for i, (m, n) in enumerate(shapes):
        dy = (rnd(rows, m, seed=seed + 3 * i) * torch.exp(rnd(1, m, seed=seed + 7))).to(tdt(code)).float()
        x = rnd(rows, n, seed=seed + 3 * i + 1) * torch.exp(2 * rnd(rows, n // 32, seed=seed + 9)).repeat_interleave(32, 1)
        c, s = q8_plain(x.to(tdt(code)))
        out.append((dy, q8_restore(c, s), sliced(dy, pad, code), c.to(torch.int8).cuda(), (torch.log2(s) + 127).to(torch.uint8).cuda()))
    return out


@pytest.mark.parametrize('code', DTYPES)
@pytest.mark.parametrize('rows,shapes,pad', WG_CASES)
def test_wgrad(K, code, rows, shapes, pad):
    ins = packed_inputs(rows, shapes, code, seed=rows, pad=pad)
    need = K.wgrad_packed_ws_bytes([(m, n, rows) for m, n in shapes], code)
    ws = torch.full((max(4, need // 4),), float('nan'), device='cuda')
    base = [rnd(m, n, seed=50 + i) for i, (m, n) in enumerate(shapes)]
    outs = [b.cuda() for b in base]
    K.wgrad_packed([(d, c, s, o) for (_, _, d, c, s), o in zip(ins, outs)], code, ws)
    fresh = [torch.full_like(o, float('nan')) for o in outs]
    K.wgrad_packed([(d, c, s, o) for (_, _, d, c, s), o in zip(ins, fresh)], code, ws, accumulate=False)
    for i, (dy, x, _, _, _) in enumerate(ins):
        ref, mag = dy.double().t() @ x, dy.double().abs().t() @ x.abs()
        # every product is exact (bf16) or off by u; rows + 16 additions, each off by at most 2 u of the magnitudes so far
        tol = 2 * (rows + 16) * U * mag
        within(fresh[i], ref, tol, f'dW {i}')
        within(outs[i], base[i].double() + ref, tol + 2 * U * (base[i].double().abs() + ref.abs()), f'dW {i} added')
    again = [torch.empty_like(o) for o in outs]
    K.wgrad_packed([(d, c, s, o) for (_, _, d, c, s), o in zip(ins, again)], code, ws, accumulate=False)
    assert all(torch.equal(a, b) for a, b in zip(again, fresh))                   # the same bits each time


# sizes at which each tile is chosen, ragged at both edges and in the rows: 256 x 256 whole and in ranges, 256 x 128 whole and in ranges,
# 128 x 128 whole and in ranges, 64 x 64 whole and in ranges, with odd and even numbers of its steps of 128 rows
LARGE_CASES = [(65, [(4104, 2080)]), (130, [(776, 3104)] * 3), (8199, [(2056, 2080)]), (8199, [(2056, 2080)] * 2), (130, [(4104, 288)] * 3), (4099, [(3080, 288)]), (2050, [(264, 288)] * 3),
               (4099, [(1032, 1056)]), (1100, [(1032, 1056)] * 2), (4099, [(1288, 800)]), (128, [(64, 64)]), (129, [(72, 96)]), (256, [(200, 224)]), (300, [(1032, 1056)]),
               (641, [(72, 32), (520, 416)]), (1025, [(2312, 800)]), (6001, [(200, 224)] * 2), (8199, [(776, 800)])]


# fp32: one step, odd and even numbers of steps, one and several ranges, ragged at both edges and in the rows
F32_CASES = [(64, [(64, 64)]), (65, [(72, 96)]), (129, [(72, 32), (8, 160)]), (577, [(200, 224)]), (2307, [(520, 416)]), (4099, [(776, 800)]), (1025, [(264, 288)] * 3)]


@pytest.mark.parametrize('code,rows,shapes', [(1, *c) for c in LARGE_CASES] + [(0, *c) for c in F32_CASES])
def test_wgrad_tiles(K, code, rows, shapes):
    gen = torch.Generator(device='cuda').manual_seed(rows)
    need = K.wgrad_packed_ws_bytes([(m, n, rows) for m, n in shapes], code)
    ws = torch.full((max(4, need // 4),), float('nan'), device='cuda')
    probs, refs = [], []
    for m, n in shapes:
        dy = torch.randn(rows, m + 8, device='cuda', generator=gen).to(tdt(code))[:, 8:]
        x = torch.randn(rows, n, device='cuda', generator=gen).to(tdt(code))
        c, s = torch.empty(rows, n, device='cuda', dtype=torch.int8), torch.empty(rows, n // 32, device='cuda', dtype=torch.uint8)
        K.act_pack(x, c, s, code)
        probs.append((dy, c, s, torch.full((m, n), float('nan'), device='cuda')))
        xd = c.double() * torch.exp2(s.double() - 127).repeat_interleave(32, 1)
        dt = dy.double().t().contiguous()
        refs.append((dt @ xd, dt.abs() @ xd.abs()))
    K.wgrad_packed(probs, code, ws, accumulate=False)
    for (dy, c, s, out), (ref, mag) in zip(probs, refs):
        within(out, ref.cpu(), 2 * (rows + 16) * U * mag.cpu(), 'dW')
        # a lost step would still be inside the worst case of thousands of additions; their errors are independent and each at most u of a
        # partial sum, which is below mag: eight times their root mean square
        assert float(((out.double() - ref).abs() / mag).max()) <= 8 * U * rows ** 0.5 + 8 * U
    K.wgrad_packed(probs, code, ws)
    for (dy, c, s, out), (ref, mag) in zip(probs, refs):
        within(out, 2 * ref.cpu(), (4 * (rows + 16) * U * mag + 4 * U * ref.abs()).cpu(), 'dW added')


@pytest.mark.parametrize('code', DTYPES)
def test_wgrad_passes_nan_groups_on(K, code):
    rows, m, n = 70, 16, 96
    (dy, x, d, c, s), = packed_inputs(rows, [(m, n)], code, seed=3)
    s[69, 1] = 255
    out = torch.zeros(m, n, device='cuda')
    ws = torch.empty(max(16, K.wgrad_packed_ws_bytes([(m, n, rows)], code)), device='cuda', dtype=torch.uint8)
    K.wgrad_packed([(d, c, s, out)], code, ws)
    assert bool(out[:, 32:64].isnan().all()) and bool(out[:, :32].isfinite().all()) and bool(out[:, 64:].isfinite().all())


@pytest.mark.parametrize('code', DTYPES)
def test_no_rows(K, code):
    t = tdt(code)
    e = lambda *s, dtype=t: torch.empty(*s, device='cuda', dtype=dtype)          # noqa: E731
    K.act_pack(e(0, 64), e(0, 64, dtype=torch.int8), e(0, 2, dtype=torch.uint8), code)
    K.act_unpack(e(0, 64, dtype=torch.int8), e(0, 2, dtype=torch.uint8), e(0, 64), code)
    g = torch.ones(64, device='cuda')
    K.qk_norm_rope_fwd(e(0, 128), e(0, 128), 1, 1, code, gq=g, gk=g)
    dgq, dgk = torch.ones(64, device='cuda'), torch.ones(64, device='cuda')
    K.qk_norm_rope_bwd(e(0, 128), e(0, 128), 1, 1, code, x=e(0, 128), gq=g, gk=g, dgq=dgq, dgk=dgk)
    assert bool((dgq == 1).all())
    K.qk_norm_rope_bwd(e(0, 128), e(0, 128), 1, 1, code, x=e(0, 128), gq=g, gk=g, dgq=dgq, dgk=dgk, accumulate=False)
    assert bool((dgq == 0).all()) and bool((dgk == 0).all())
    out = torch.ones(8, 32, device='cuda')
    pr = [(e(0, 8), e(0, 32, dtype=torch.int8), e(0, 1, dtype=torch.uint8), out)]
    K.wgrad_packed(pr, code)
    assert bool((out == 1).all())
    K.wgrad_packed(pr, code, accumulate=False)
    assert bool((out == 0).all())


# ------------------------------------------------------------------------------------------------------------- together, streams, graphs
def _chain(K, st, code):
    """what a training step makes of them: norm + rotation with a checkpoint, another activation put away, both backward passes"""
    K.qk_norm_rope_fwd(st['x'], st['y'], 4, 4, code, packed=st['pk'], **st['par'])
    K.act_pack(st['a'], *st['pa'], code)
    K.qk_norm_rope_bwd(st['dy'], st['dx'], 4, 4, code, packed=st['pk'], dgq=st['dgq'], dgk=st['dgk'], ws=st['ws'], accumulate=False, **st['par'])
    K.wgrad_packed([(st['dx'], *st['pa'], st['dw'])], code, st['wsw'], accumulate=False)
    K.act_unpack(*st['pa'], st['ar'], code)


def _chain_state(K, code, seed):
    rows, C, t = 4 * 65, 512, tdt(code)
    e = lambda *s, dtype=t: torch.empty(*s, device='cuda', dtype=dtype)          # noqa: E731
    cos, sin = tables(65)
    return dict(x=rnd(rows, C, seed=seed).to(t).cuda(), a=rnd(rows, 320, seed=seed + 1).to(t).cuda(), dy=rnd(rows, C, seed=seed + 2).to(t).cuda(),
                y=e(rows, C), dx=e(rows, C), ar=e(rows, 320), dw=e(C, 320, dtype=torch.float32), dgq=e(64, dtype=torch.float32),
                dgk=e(64, dtype=torch.float32), pk=(e(rows, C, dtype=torch.int8), e(rows, C // 32, dtype=torch.uint8)),
                pa=(e(rows, 320, dtype=torch.int8), e(rows, 10, dtype=torch.uint8)),
                ws=e(K.qk_norm_rope_ws_bytes(rows, 4, 4), dtype=torch.uint8), wsw=e(max(16, K.wgrad_packed_ws_bytes([(C, 320, rows)], code)), dtype=torch.uint8),
                par=dict(gq=torch.rand(64).cuda() + 0.5, gk=torch.rand(64).cuda() + 0.5, cos=cos.cuda(), sin=sin.cuda(), eps=1e-6))


OUTS = ('y', 'dx', 'ar', 'dw', 'dgq', 'dgk')


@pytest.mark.parametrize('code', DTYPES)
def test_chain_on_streams(K, code):
    """two chains side by side on streams of their own give what they give alone"""
    a, b = _chain_state(K, code, 1), _chain_state(K, code, 100)
    for st in (a, b):
        _chain(K, st, code)
    torch.cuda.synchronize()
    want = [{k: st[k].clone() for k in OUTS} for st in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for st in (a, b):
            for k in OUTS:
                st[k].zero_()
        torch.cuda.synchronize()
        for s, st in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                _chain(K, st, code)
        torch.cuda.synchronize()
        for w, st in zip(want, (a, b)):
            for k in OUTS:
                assert torch.equal(w[k], st[k]), k


@pytest.mark.parametrize('code', DTYPES)
def test_chain_in_a_graph(K, code):
    """captured once, replayed over changing inputs with eager work in between"""
    st = _chain_state(K, code, 7)
    _chain(K, st, code)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _chain(K, st, code)
    for i in range(4):
        new = _chain_state(K, code, 200 + 10 * i)
        for k in ('x', 'a', 'dy'):
            st[k].copy_(new[k])
        for k in ('gq', 'gk'):
            st['par'][k].copy_(new['par'][k])
        _chain(K, new, code)
        g.replay()
        torch.cuda.synchronize()
        for k in OUTS:
            assert torch.equal(new[k], st[k]), (i, k)


# ------------------------------------------------------------------------------------------------------------- far ends of the calls
@pytest.mark.parametrize('code', DTYPES)
def test_offsets_beyond_32_bits(K, code):
    """slices of a buffer whose last rows lie more than 2^32 elements behind the first"""
    rows, ld, t = 70001, 65536, tdt(code)
    buf = torch.empty(rows, ld, device='cuda', dtype=t)
    pick = torch.tensor([0, 1, 32767, 32768, 65535, 65536, rows - 2, rows - 1], device='cuda')
    x, y = buf[:, 64:64 + 256], buf[:, 1024:1024 + 256]
    x.copy_(torch.randn(rows, 256, device='cuda', generator=torch.Generator(device='cuda').manual_seed(1)).to(t))
    g = [torch.rand(64, device='cuda') + 0.5 for _ in range(2)]
    codes, scales = torch.empty(rows, 256, device='cuda', dtype=torch.int8), torch.empty(rows, 8, device='cuda', dtype=torch.uint8)
    K.qk_norm_rope_fwd(x, y, 2, 2, code, gq=g[0], gk=g[1], packed=(codes, scales))
    few = x[pick].contiguous()
    ref = torch.empty_like(few)
    c2, s2 = torch.empty(len(pick), 256, device='cuda', dtype=torch.int8), torch.empty(len(pick), 8, device='cuda', dtype=torch.uint8)
    K.qk_norm_rope_fwd(few, ref, 2, 2, code, gq=g[0], gk=g[1], packed=(c2, s2))
    assert torch.equal(y[pick], ref) and torch.equal(codes[pick], c2) and torch.equal(scales[pick], s2)
    K.act_pack(x, codes, scales, code)
    assert torch.equal(codes[pick], c2) and torch.equal(scales[pick], s2)
    K.act_unpack(codes, scales, y, code)
    r2 = torch.empty_like(few)
    K.act_unpack(c2, s2, r2, code)
    assert torch.equal(y[pick], r2)
    dx = torch.empty(rows, 256, device='cuda', dtype=t)
    dg = [torch.empty(64, device='cuda') for _ in range(4)]
    ws = torch.empty(K.qk_norm_rope_ws_bytes(rows, 2, 2), device='cuda', dtype=torch.uint8)
    kw = dict(gq=g[0], gk=g[1], accumulate=False, ws=ws)
    K.qk_norm_rope_bwd(x, dx, 2, 2, code, x=x, dgq=dg[0], dgk=dg[1], **kw)
    d2 = torch.empty_like(few)
    K.qk_norm_rope_bwd(few, d2, 2, 2, code, x=few, dgq=dg[2], dgk=dg[3], **kw)
    assert torch.equal(dx[pick], d2)
    # weight gradients: everything but the picked rows is zero, so the sums are those of the picked rows
    dy = buf[:, 2048:2048 + 64]
    dy.zero_()
    some = torch.randn(len(pick), 64, device='cuda', generator=torch.Generator(device='cuda').manual_seed(2)).to(t)
    dy[pick] = some
    outs = [torch.empty(64, 256, device='cuda') for _ in range(2)]
    wsw = torch.empty(max(16, K.wgrad_packed_ws_bytes([(64, 256, rows)], code)), device='cuda', dtype=torch.uint8)
    K.wgrad_packed([(dy, codes, scales, outs[0])], code, wsw, accumulate=False)
    x64 = r2.cpu().double()
    want, mag = some.cpu().double().t() @ x64, some.cpu().double().abs().t() @ x64.abs()
    within(outs[0], want, 2 * (len(pick) + 80) * U * mag, 'dW')


@pytest.mark.parametrize('code', DTYPES)
def test_one_long_row_set_of_codes(K, code):
    """more than 2^31 values in one contiguous tensor"""
    rows, C, t = 66000, 32768 + 32, tdt(code)
    assert rows * C > 2 ** 31
    x = torch.zeros(rows, C, device='cuda', dtype=t)
    pick = torch.tensor([0, 1, 32000, 65000, rows - 1], device='cuda')
    few = torch.randn(len(pick), C, device='cuda', generator=torch.Generator(device='cuda').manual_seed(3)).to(t)
    x[pick] = few
    codes, scales = torch.empty(rows, C, device='cuda', dtype=torch.int8), torch.empty(rows, C // 32, device='cuda', dtype=torch.uint8)
    K.act_pack(x, codes, scales, code)
    c2, s2 = torch.empty(len(pick), C, device='cuda', dtype=torch.int8), torch.empty(len(pick), C // 32, device='cuda', dtype=torch.uint8)
    K.act_pack(few, c2, s2, code)
    assert torch.equal(codes[pick], c2) and torch.equal(scales[pick], s2)
    K.act_unpack(codes, scales, x, code)
    r2 = torch.empty_like(few)
    K.act_unpack(c2, s2, r2, code)
    assert torch.equal(x[pick], r2)


@pytest.mark.parametrize('code', DTYPES)
def test_nan_and_infinity_stay_in_their_head(K, code):
    case = (1, 6, 3, 2, True, True, False, 0)
    x, dy, gq, gk, cos, sin = qk_inputs(case, code, seed=70)
    bad = x.clone()
    bad[2, 64 + 5] = float('nan')
    bad[4, 3 * 64 + 40] = float('inf')
    hit = torch.zeros(6, 5, dtype=torch.bool)
    hit[2, 1] = hit[4, 3] = True
    par = dict(gq=cu(gq), gk=cu(gk), cos=cu(cos), sin=cu(sin), eps=1e-6)
    ys, dxs = [], []
    ws = torch.empty(K.qk_norm_rope_ws_bytes(6, 3, 2), device='cuda', dtype=torch.uint8)
    for v in (x, bad):
        v = v.to(tdt(code)).cuda()
        y, dx = torch.empty_like(v), torch.empty_like(v)
        pk = (torch.empty(6, 320, device='cuda', dtype=torch.int8), torch.empty(6, 10, device='cuda', dtype=torch.uint8))
        K.qk_norm_rope_fwd(v, y, 3, 2, code, packed=pk, **par)
        dg = [torch.zeros(64, device='cuda') for _ in range(2)]
        K.qk_norm_rope_bwd(dy.to(tdt(code)).cuda(), dx, 3, 2, code, packed=pk, dgq=dg[0], dgk=dg[1], ws=ws, **par)
        ys.append(y.cpu().reshape(6, 5, 64)); dxs.append(dx.cpu().reshape(6, 5, 64))
    for a, b in (ys, dxs):
        assert torch.equal(a[~hit], b[~hit])
        assert bool(b[hit].isnan().any(-1).all())


@pytest.mark.parametrize('code', DTYPES)
def test_rows_behind_the_last_stay(K, code):
    t = tdt(code)
    big = torch.full((9, 256), 3.0, device='cuda', dtype=t)
    x = rnd(5, 256, seed=1).to(t).cuda()
    g = torch.ones(64, device='cuda')
    K.qk_norm_rope_fwd(x, big[:5], 2, 2, code, gq=g, gk=g)
    assert bool((big[5:] == 3).all()) and not bool((big[:5] == 3).any())
    dg = [torch.zeros(64, device='cuda') for _ in range(2)]
    big.fill_(3.0)
    K.qk_norm_rope_bwd(x, big[:5], 2, 2, code, x=x, gq=g, gk=g, dgq=dg[0], dgk=dg[1],
                       ws=torch.empty(K.qk_norm_rope_ws_bytes(5, 2, 2), device='cuda', dtype=torch.uint8))
    assert bool((big[5:] == 3).all())


@pytest.mark.parametrize('code', DTYPES)
def test_two_graphs_share_their_workspaces(K, code):
    a, b = _chain_state(K, code, 11), _chain_state(K, code, 12)
    b['ws'], b['wsw'] = a['ws'], a['wsw']
    graphs = []
    for st in (a, b):
        _chain(K, st, code)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            _chain(K, st, code)
        graphs.append(g)
    want = []
    for st in (a, b):
        _chain(K, st, code)
        torch.cuda.synchronize()
        want.append({k: st[k].clone() for k in OUTS})
    for _ in range(3):
        for st in (a, b):
            for k in OUTS:
                st[k].zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for w, st in zip(want, (a, b)):
            for k in OUTS:
                assert torch.equal(w[k], st[k]), k


def test_refusals_on_the_device(K):
    """what only device tensors reach: overlapping arguments, strides and alignments the kernels do not take, short workspaces"""
    from s4former_amd._lib import S4FError
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, device='cuda', dtype=dtype)                      # noqa: E731
    g, buf = z(64), z(9, 400)
    i8, u8 = lambda *s: z(*s, dtype=torch.int8), lambda *s: z(*s, dtype=torch.uint8)                     # noqa: E731
    flat = z(4096)
    out = z(16, 64)
    ok = (z(200, 8), i8(200, 64), u8(200, 2))
    for what, call in {
        'partly overlapping x and y': lambda: K.qk_norm_rope_fwd(buf[:4, :128], buf[:4, 64:192], 1, 1, 0, gq=g, gk=g),
        'shifted rows': lambda: K.qk_norm_rope_fwd(buf[:4, :128], buf[1:5, :128], 1, 1, 0, gq=g, gk=g),
        'misaligned columns': lambda: K.qk_norm_rope_fwd(buf[:4, 1:129], z(4, 128), 1, 1, 0, gq=g, gk=g),
        'misaligned row stride': lambda: K.act_pack(z(4, 66)[:, :64], i8(4, 64), u8(4, 2), 0),
        'elements of a row apart': lambda: K.act_pack(z(4, 128)[:, ::2], i8(4, 64), u8(4, 2), 0),
        'transposed': lambda: K.act_pack(z(64, 64).t(), i8(64, 64), u8(64, 2), 0),
        'rows of y overlap': lambda: K.act_unpack(i8(4, 64), u8(4, 2), flat.as_strided((4, 64), (16, 1)), 0),
        'codes of another size': lambda: K.act_pack(z(4, 64), i8(5, 64), u8(4, 2), 0),
        'codes of another type': lambda: K.act_pack(z(4, 64), u8(4, 64), u8(4, 2), 0),
        'codes with gaps': lambda: K.act_pack(z(4, 64), i8(4, 128)[:, :64], u8(4, 2), 0),
        'tables that do not divide the rows': lambda: K.qk_norm_rope_fwd(z(4, 128), z(4, 128), 1, 1, 0, cos=z(3, 32), sin=z(3, 32)),
        'tables of another width': lambda: K.qk_norm_rope_fwd(z(4, 128), z(4, 128), 1, 1, 0, cos=z(4, 64), sin=z(4, 64)),
        'tables of different lengths': lambda: K.qk_norm_rope_fwd(z(4, 128), z(4, 128), 1, 1, 0, cos=z(4, 32), sin=z(2, 32)),
        'half a norm': lambda: K.qk_norm_rope_fwd(z(4, 128), z(4, 128), 1, 1, 0, gq=g),
        'gains in another type': lambda: K.qk_norm_rope_fwd(z(4, 128), z(4, 128), 1, 1, 0, gq=g.bfloat16(), gk=g.bfloat16()),
        'checkpoint without the norm': lambda: K.qk_norm_rope_fwd(z(4, 128), z(4, 128), 1, 1, 0, cos=z(4, 32), sin=z(4, 32), packed=(i8(4, 128), u8(4, 4))),
        'no workspace': lambda: K.qk_norm_rope_bwd(z(4, 128), z(4, 128), 1, 1, 0, x=z(4, 128), gq=g, gk=g, dgq=z(64), dgk=z(64)),
        'one gain gradient for both': lambda: K.qk_norm_rope_bwd(z(4, 128), z(4, 128), 1, 1, 0, x=z(4, 128), gq=g, gk=g, dgq=g, dgk=g, ws=z(4096)),
        'x and its checkpoint': lambda: K.qk_norm_rope_bwd(z(4, 128), z(4, 128), 1, 1, 0, x=z(4, 128), packed=(i8(4, 128), u8(4, 4)), gq=g, gk=g, dgq=z(64),
                                                           dgk=z(64), ws=z(4096)),
        'one output twice': lambda: K.wgrad_packed([(z(200, 16), *ok[1:], out), (z(200, 16), *ok[1:], out)], 0, z(1 << 16)),
        'outputs that overlap': lambda: K.wgrad_packed([(z(200, 8), *ok[1:], out[:8]), (z(200, 16), *ok[1:], out)], 0, z(1 << 16)),
        'output in the workspace': lambda: K.wgrad_packed([(*ok, flat[:512].view(8, 64))], 0, flat),
        'broadcast rows of dy': lambda: K.wgrad_packed([(z(1, 8).expand(200, 8), *ok[1:], z(8, 64))], 0, z(1 << 16)),
        'short workspace': lambda: K.wgrad_packed([(z(4000, 64), i8(4000, 64), u8(4000, 2), z(64, 64))], 0, z(4)),
    }.items():
        with pytest.raises(S4FError):
            call()
            pytest.fail(f'not refused: {what}')
