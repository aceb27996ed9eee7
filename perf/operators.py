"""Cases for the operators of the encoder layer's training options: the norm of queries and keys with the position rotation, and
activation checkpoints in 8 bits with the weight gradients that read them.

kinds of a case
  qk_fwd   queries and keys of a packed projection [rows, (Hq + 2 Hk) 64]: RMS norm per head (gains shared by the heads of a kind),
           rotation of the pair (i, i + 32) of a head by the angle of the row's position
  qk_bwd   its backward from the saved queries and keys: their gradient, and the gradients of the two gains
  qk_step  both as a training step has them, with the pre-norm queries and keys kept as an 8-bit checkpoint in between
  ckpt     an activation put away in 8 bits and restored: groups of 32 channels of a row share a power-of-two scale
  wgrad    weight gradients dW = dY^T X of up to four linear layers whose inputs X are 8-bit checkpoints

`own` false: elementary torch operations in 32 bits, rounded once at the end; `own` true: the calls of s4former_amd.kernels.
"""
import math

import torch

own = False

GROUP = 32          # channels that share a scale
HEAD = 64           # head dimension
EPS = 1e-6


# ------------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one 512 x 512 image through a 12-head backbone at inference: 32 x 32 patches + cls
        dict(name='qk_fwd_image', kind='qk_fwd', dtype='bf16', B=1, N=1025, Hq=12, Hk=12, norm=True, rope=True, tab='shared'),
        # the rotation alone for the tokens of a small crop, in 32 bits (the smallest call: latency)
        dict(name='qk_fwd_crop_f32', kind='qk_fwd', dtype='f32', B=2, N=17, Hq=4, Hk=4, norm=False, rope=True, tab='shared'),
        # the teacher's pass over the step's 16 images, each with positions of its own crop
        dict(name='qk_fwd_batch', kind='qk_fwd', dtype='bf16', B=16, N=1025, Hq=12, Hk=12, norm=True, rope=True, tab='per_image'),
        # backward on three 768 x 768 images (48 x 48 patches + cls), 16 query heads over 4 key heads
        dict(name='qk_bwd_shared_heads', kind='qk_bwd', dtype='bf16', B=3, N=2305, Hq=16, Hk=4, norm=True, rope=True, tab='shared'),
        # the student's 16 images: forward, 8-bit checkpoint, backward from it
        dict(name='qk_step_batch', kind='qk_step', dtype='bf16', B=16, N=1025, Hq=12, Hk=12, norm=True, rope=True, tab='shared'),
        # the input of one image's attention block
        dict(name='ckpt_image_f32', kind='ckpt', dtype='f32', rows=1025, C=768, pad=0, act='ln'),
        # the hidden activation of a wide feed-forward block on 8 images
        dict(name='ckpt_hidden', kind='ckpt', dtype='bf16', rows=8200, C=4096, pad=0, act='gelu'),
        # a narrow slice of a wider buffer, rows of ragged images
        dict(name='ckpt_slice', kind='ckpt', dtype='bf16', rows=6919, C=352, pad=1184, act='gauss'),
        # the output projection's weights from one image
        dict(name='wgrad_proj_image', kind='wgrad', dtype='bf16', rows=1025, shapes='768x768'),
        # the packed query / key / value projection's weights from the step's 16 images
        dict(name='wgrad_qkv_batch', kind='wgrad', dtype='bf16', rows=16400, shapes='2304x768'),
        # the four weight gradients of a wide encoder layer at once, 8 images
        dict(name='wgrad_layer', kind='wgrad', dtype='bf16', rows=8200, shapes='4096x1024,1024x4096,1024x1024,1024x1024'),
        # 32-bit mode, ragged sizes
        dict(name='wgrad_ragged_f32', kind='wgrad', dtype='f32', rows=2307, shapes='520x416'),
    ]


def _spread(rng, lo, hi):
    """a whole number spread over [lo, hi] by its logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(['qk_fwd', 'qk_bwd', 'qk_step', 'ckpt', 'ckpt', 'wgrad', 'wgrad'])
    dtype = rng.choice(['bf16', 'bf16', 'f32'])
    if kind.startswith('qk'):
        hk = rng.choice([1, 2, 3, 4, 6, 12, 16])
        hq = hk * rng.choice([1, 1, 2, 4]) if hk <= 4 else hk
        norm, rope = rng.choice([(True, True), (True, True), (True, False), (False, True)])
        norm = norm or kind == 'qk_step'                     # nothing is put away for the rotation alone
        n = _spread(rng, 1, 2500)
        b = _spread(rng, 1, max(1, min(16, 16400 // n)))
        return dict(kind=kind, dtype=dtype, B=b, N=n, Hq=hq, Hk=hk, norm=norm, rope=rope, tab=rng.choice(['shared', 'per_image']))
    if kind == 'ckpt':
        rows = _spread(rng, 1, 16400)
        c = GROUP * _spread(rng, 1, 128)
        while rows * c > 8200 * 4096:
            c = max(GROUP, c // 2 // GROUP * GROUP)
        return dict(kind=kind, dtype=dtype, rows=rows, C=c, pad=rng.choice([0, 0, 8, 640]), act=rng.choice(['ln', 'gelu', 'gauss']))
    rows = _spread(rng, 1, 16400)
    shapes = []
    for _ in range(rng.choice([1, 1, 2, 4])):
        m, n = 8 * _spread(rng, 1, 512), GROUP * _spread(rng, 1, 128)
        if dtype == 'f32':
            m, n = min(m, 1024), min(n, 1024)
        while rows * m * n > 8200 * 1024 * 4096 // 4:
            m = max(8, m // 2 // 8 * 8)
        shapes.append('%dx%d' % (m, n))
    return dict(kind=kind, dtype=dtype, rows=rows, shapes=','.join(shapes))


# ------------------------------------------------------------------------------------------------------------------ inputs
def _type(case):
    return torch.bfloat16 if case['dtype'] == 'bf16' else torch.float32


def _shapes(case):
    return [tuple(int(v) for v in s.split('x')) for s in case['shapes'].split(',')]


def _randn(gen, *shape):
    return torch.randn(*shape, device='cuda', generator=gen)


def _activation(gen, rows, c, act):
    """what the layers put away: normalised tokens with a few strong channels, GELU outputs, attention outputs"""
    x = _randn(gen, rows, c)
    if act == 'ln':
        strong = torch.rand(c, device='cuda', generator=gen) < 0.02
        return x * torch.where(strong, 12.0, 1.0)
    if act == 'gelu':
        return 0.5 * x * (1.0 + torch.erf(x * 0.7071067811865476))
    return 0.3 * x


def _tables(case, gen):
    """cos and sin [P, 32] of the positions: the rows and columns of a patch grid, 16 frequencies each, the first token unrotated;
    for positions of its own every image has an offset"""
    n, b = case['N'], (case['B'] if case['tab'] == 'per_image' else 1)
    w = max(1, int(math.isqrt(max(1, n - 1))))
    idx = torch.arange(n, device='cuda', dtype=torch.float64) - 1
    yy, xx = torch.div(idx, w, rounding_mode='floor'), torch.remainder(idx, w)
    freq = 100.0 ** (-torch.arange(16, device='cuda', dtype=torch.float64) / 16)
    off = torch.floor(torch.rand(b, 2, device='cuda', generator=gen).double() * 64) if case['tab'] == 'per_image' else torch.zeros(1, 2, device='cuda').double()
    ang = torch.cat([(yy[None, :, None] + off[:, 0, None, None]) * freq, (xx[None, :, None] + off[:, 1, None, None]) * freq], -1)
    ang[:, 0] = 0
    ang = ang.reshape(b * n, 32)
    return ang.cos().float(), ang.sin().float()


def _put_away(x):
    """(codes int8, scales uint8) of a 32-bit tensor [rows, C]: code = round(x / s), s the least power of two that keeps |code| <= 127"""
    g = x.reshape(x.shape[0], -1, GROUP)
    m, e = torch.frexp(g.abs().amax(-1))                     # amax = m 2^e, m in [0.5, 1)
    e = torch.clamp(e - 7 + (m >= 255.0 / 256.0).to(e.dtype), min=-126)
    codes = torch.round(torch.ldexp(g, -e[..., None]))
    return codes.to(torch.int8).reshape(x.shape), (e + 127).to(torch.uint8)


def _restored(codes, scales):
    g = codes.float().reshape(codes.shape[0], -1, GROUP)
    return torch.ldexp(g, scales.to(torch.int32)[..., None] - 127).reshape(codes.shape)


def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    kind, t = case['kind'], _type(case)
    st = dict(case=case)
    if own:
        from s4former_amd import kernels as K
        st['code'] = K.BF16 if t == torch.bfloat16 else K.F32
    if kind.startswith('qk'):
        rows, hq, hk = case['B'] * case['N'], case['Hq'], case['Hk']
        width = (hq + hk) * HEAD
        scale = torch.exp(0.3 * _randn(gen, 1, width + hk * HEAD))
        st['qkv'] = (_randn(gen, rows, width + hk * HEAD) * scale).to(t)
        st['x'] = st['qkv'][:, :width]
        st['gq'] = 1 + 0.1 * _randn(gen, HEAD) if case['norm'] else None
        st['gk'] = 1 + 0.1 * _randn(gen, HEAD) if case['norm'] else None
        st['cos'], st['sin'] = _tables(case, gen) if case['rope'] else (None, None)
        st['y'] = torch.empty_like(st['qkv'])[:, :width]     # the packed buffer that attention reads; its values are there already
        if kind != 'qk_fwd':
            st['dqkv'] = (0.02 * _randn(gen, rows, width + hk * HEAD)).to(t)
            st['dy'] = st['dqkv'][:, :width]
            if own:
                st['dx'] = torch.empty(rows, width, device='cuda', dtype=t)
                st['dgq'], st['dgk'] = (torch.empty(HEAD, device='cuda'), torch.empty(HEAD, device='cuda')) if case['norm'] else (None, None)
                st['ws'] = torch.empty(K.qk_norm_rope_ws_bytes(rows, hq, hk), device='cuda', dtype=torch.uint8)
                if kind == 'qk_step':
                    st['codes'] = torch.empty(rows, width, device='cuda', dtype=torch.int8)
                    st['scales'] = torch.empty(rows, width // GROUP, device='cuda', dtype=torch.uint8)
    elif kind == 'ckpt':
        rows, c, pad = case['rows'], case['C'], case['pad']
        buf = torch.zeros(rows, c + pad, device='cuda', dtype=t)
        buf[:, :c] = _activation(gen, rows, c, case['act']).to(t)
        st['x'] = buf[:, :c]
        if own:
            st['codes'] = torch.empty(rows, c, device='cuda', dtype=torch.int8)
            st['scales'] = torch.empty(rows, c // GROUP, device='cuda', dtype=torch.uint8)
            st['y'] = torch.empty(rows, c, device='cuda', dtype=t)
    else:
        st['dy'], st['codes'], st['scales'], st['out'] = [], [], [], []
        for i, (m, n) in enumerate(_shapes(case)):
            st['dy'].append((0.02 * _randn(gen, case['rows'], m)).to(t))
            c, s = _put_away(_activation(gen, case['rows'], n, ('ln', 'gelu', 'ln', 'gauss')[i % 4]).to(t).float())
            st['codes'].append(c)
            st['scales'].append(s)
            st['out'].append(torch.empty(m, n, device='cuda'))
        if own:
            st['ws'] = torch.empty(K.wgrad_packed_ws_bytes([(m, n, case['rows']) for m, n in _shapes(case)], st['code']),
                                   device='cuda', dtype=torch.uint8)
    return st


# ------------------------------------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    from s4former_amd import kernels as K
    case, code = st['case'], st['code']
    kind = case['kind']
    if kind == 'ckpt':
        K.act_pack(st['x'], st['codes'], st['scales'], code)
        K.act_unpack(st['codes'], st['scales'], st['y'], code)
        return st['y']
    if kind == 'wgrad':
        K.wgrad_packed([(st['dy'][i], st['codes'][i], st['scales'][i], st['out'][i]) for i in range(len(st['out']))], code, st['ws'],
                       accumulate=False)
        return st['out']
    hq, hk = case['Hq'], case['Hk']
    par = dict(gq=st['gq'], gk=st['gk'], cos=st['cos'], sin=st['sin'], eps=EPS)
    if kind == 'qk_fwd':
        K.qk_norm_rope_fwd(st['x'], st['y'], hq, hk, code, **par)
        return st['y']
    grads = dict(dgq=st['dgq'], dgk=st['dgk'], ws=st['ws'], accumulate=False)
    if kind == 'qk_bwd':
        K.qk_norm_rope_bwd(st['dy'], st['dx'], hq, hk, code, x=st['x'], **par, **grads)
        return (st['dx'], st['dgq'], st['dgk']) if case['norm'] else (st['dx'],)
    packed = (st['codes'], st['scales'])
    K.qk_norm_rope_fwd(st['x'], st['y'], hq, hk, code, packed=packed, **par)
    K.qk_norm_rope_bwd(st['dy'], st['dx'], hq, hk, code, packed=packed, **par, **grads)
    return (st['y'], st['dx'], st['dgq'], st['dgk']) if case['norm'] else (st['y'], st['dx'])


def _gains(st, case):
    return torch.cat([st['gq'].expand(case['Hq'], HEAD), st['gk'].expand(case['Hk'], HEAD)]) if case['norm'] else None


def _turn(lo, hi, st, case, sign):
    """the pairs (lo, hi) [rows, H, 32] turned by sign * the angle of their row"""
    if not case['rope']:
        return torch.cat([lo, hi], -1)
    p = st['cos'].shape[0]
    shape = (-1, p) + tuple(lo.shape[1:])
    c, s = st['cos'][None, :, None, :], sign * st['sin'][None, :, None, :]
    a, b = lo.reshape(shape), hi.reshape(shape)
    return torch.cat([a * c - b * s, b * c + a * s], -1).reshape(lo.shape[0], lo.shape[1], HEAD)


def _plain_fwd(st, case):
    x = st['x'].float().reshape(-1, case['Hq'] + case['Hk'], HEAD)
    if case['norm']:
        x = x * (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * _gains(st, case)
    y = _turn(x[..., :32], x[..., 32:], st, case, 1.0)
    return y.reshape(st['x'].shape).to(st['x'].dtype)


def _plain_bwd(st, case, x):
    hq, h = case['Hq'], case['Hq'] + case['Hk']
    dy = st['dy'].float().reshape(-1, h, HEAD)
    dz = _turn(dy[..., :32], dy[..., 32:], st, case, -1.0)
    if not case['norm']:
        return (dz.reshape(st['x'].shape).to(st['x'].dtype),)
    x = x.reshape(-1, h, HEAD)
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    u = x * r
    du = dz * _gains(st, case)
    dx = r * (du - u * (du * u).mean(-1, keepdim=True))
    dg = (dz * u).sum(0)
    return dx.reshape(st['x'].shape).to(st['x'].dtype), dg[:hq].sum(0), dg[hq:].sum(0)


def _run_plain(st):
    case = st['case']
    kind = case['kind']
    if kind == 'ckpt':
        return _restored(*_put_away(st['x'].float())).to(st['x'].dtype)
    if kind == 'wgrad':
        return [st['dy'][i].float().t() @ _restored(st['codes'][i], st['scales'][i]) for i in range(len(st['dy']))]
    if kind == 'qk_fwd':
        return _plain_fwd(st, case)
    if kind == 'qk_bwd':
        return _plain_bwd(st, case, st['x'].float())
    return (_plain_fwd(st, case),) + _plain_bwd(st, case, _restored(*_put_away(st['x'].float())))


# ------------------------------------------------------------------------------------------------------------------ the definition
def exact(case, seed):
    st = prepare(case, seed)
    kind = case['kind']
    if kind == 'wgrad':
        out = []
        for dy, codes, scales in zip(st['dy'], st['codes'], st['scales']):
            s = torch.exp2(scales.double() - 127)
            out.append(torch.matmul(dy.double().t().contiguous(), codes.double() * s.repeat_interleave(GROUP, 1)))
        return out

    def step(v):                                             # the scale of every value, in 64 bits
        big = v.reshape(v.shape[0], -1, GROUP).abs().max(-1).values
        e = torch.floor(torch.log2(torch.clamp(big, min=2.0 ** -200)))
        e = e + (torch.exp2(e + 1) <= big).double() - (torch.exp2(e) > big).double()          # log2 next to a power of two
        e = e - 6
        e = torch.clamp(torch.where(big / torch.exp2(e) >= 127.5, e + 1, e), min=-126)
        return torch.exp2(e).repeat_interleave(GROUP, 1)

    x = st['x'].double()
    kept = x
    if kind in ('ckpt', 'qk_step'):
        s = step(x)
        kept = torch.round(x / s) * s
    if kind == 'ckpt':
        return kept
    rows, hq, hk = x.shape[0], case['Hq'], case['Hk']
    h = hq + hk
    if case['rope']:
        turn = torch.complex(st['cos'].double(), st['sin'].double()).repeat(rows // st['cos'].shape[0], 1)[:, None]
    else:
        turn = torch.ones(rows, 1, 32, device=x.device, dtype=torch.complex128)

    def pairs(v):
        v = v.reshape(rows, h, 2, 32)
        return torch.complex(v[:, :, 0], v[:, :, 1])

    def flat(z):
        return torch.stack([z.real, z.imag], 2).reshape(rows, h * HEAD)

    def normed(v):
        v = v.reshape(rows, h, HEAD)
        r = (v.square().sum(-1, keepdim=True) / HEAD + EPS).rsqrt()
        return v * r, r

    gain = None
    if case['norm']:
        gain = torch.stack([st['gq'].double()] * hq + [st['gk'].double()] * hk)
    res = []
    if kind in ('qk_fwd', 'qk_step'):
        v = normed(x)[0] * gain if case['norm'] else x
        res.append(flat(pairs(v) * turn))
    if kind == 'qk_fwd':
        return res[0]
    back = flat(pairs(st['dy'].double()) * turn.conj())
    if not case['norm']:
        return tuple(res + [back])
    u, r = normed(kept)
    back = back.reshape(rows, h, HEAD)
    w = back * gain
    dx = (w - u * ((w * u).sum(-1, keepdim=True) / HEAD)) * r
    dg = back * u
    return tuple(res + [dx.reshape(rows, h * HEAD), dg[:, :hq].sum((0, 1)), dg[:, hq:].sum((0, 1))])


# ------------------------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    """each input read once, each output written once; a checkpoint is written and read once more, since keeping it is its purpose.
    Operations: 2 a multiply-add; a norm's square, scale and gain, a rotation's three per element."""
    ts = 2 if case['dtype'] == 'bf16' else 4
    kind = case['kind']
    if kind == 'ckpt':
        n = case['rows'] * case['C']
        return dict(bytes=n * (2 * ts + 2 + 2 / GROUP), flops=4 * n)
    if kind == 'wgrad':
        r = case['rows']
        return dict(bytes=sum(r * m * ts + r * n * (1 + 1 / GROUP) + 4 * m * n for m, n in _shapes(case)),
                    flops=sum(2 * r * m * n for m, n in _shapes(case)))
    rows = case['B'] * case['N']
    n = rows * (case['Hq'] + case['Hk']) * HEAD
    tab = (rows if case['tab'] == 'per_image' else case['N']) * 256 if case['rope'] else 0
    fwd = (4 if case['norm'] else 0) + (3 if case['rope'] else 0)
    bwd = (12 if case['norm'] else 0) + (3 if case['rope'] else 0)
    if kind == 'qk_fwd':
        return dict(bytes=2 * ts * n + tab, flops=fwd * n)
    if kind == 'qk_bwd':
        return dict(bytes=(3 if case['norm'] else 2) * ts * n + tab, flops=bwd * n)
    return dict(bytes=4 * ts * n + 2 * n * (1 + 1 / GROUP) + tab, flops=(fwd + bwd + 4) * n)
