"""The encoder layer's options (qk_norm, rope_theta, act_q8) through the public model: VisionTransformer and EncoderDecoder.

fp32 mode against 64 bits: a gradient passes at most 16 contractions of at most 1024 terms in this model, each off by at most
1024 * 2^-24 of the magnitudes it sums: 1e-3 of the tensor's largest magnitude.  bf16 mode: the framework's tolerance for one layer's
chain of bf16 roundings (2^-8 each, about eight in a row: 3e-2)."""
import pytest
import torch
import torch.nn.functional as F

import s4former_amd as S
from tests import common as C

pytestmark = pytest.mark.gpu
TOL = {'fp32': 1e-3, 'bf16': 3e-2}
EPS = 1e-6
OPT = dict(type='SGD', lr=0.001, momentum=0.9, weight_decay=0.0, paramwise_cfg=dict(custom_keys={'head': dict(lr_mult=10.)}))


@pytest.fixture(autouse=True)
def _restore_dtype():
    yield
    S.set_compute_dtype('bf16')


def make_vit(dtype, layers=2, img=64, seed=1, **flags):
    S.set_compute_dtype(dtype)
    m = S.VisionTransformer(img_size=(img, img), patch_size=16, embed_dims=256, num_layers=layers, num_heads=4, out_indices=tuple(range(layers)),
                            norm_cfg=dict(type='LN', eps=EPS), interpolate_mode='bilinear', **flags)
    g = torch.Generator().manual_seed(seed)
    for n, p in m.named_parameters():
        scale = 0.1 if n.endswith('weight') and p.dim() == 1 else 0.06
        p.data.copy_(torch.randn(p.shape, generator=g) * scale + (1.0 if n.endswith('weight') and p.dim() == 1 else 0.0))
    return m.cuda().train()


def rms(v, g):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * g


def rotate(v, hw, theta):
    """v [B, H, 1 + h w, 64]: complex pairs (i, i + 32) times exp(i angle)"""
    h, w = hw
    t = torch.arange(h * w, dtype=torch.float64)
    fr = theta ** (-torch.arange(16, dtype=torch.float64) / 16)
    ang = torch.cat([torch.div(t, w, rounding_mode='floor')[:, None] * fr, (t % w)[:, None] * fr], -1)
    ang = torch.cat([torch.zeros(1, 32, dtype=torch.float64), ang])
    z = torch.complex(v[..., :32], v[..., 32:]) * torch.polar(torch.ones_like(ang), ang)
    return torch.cat([z.real, z.imag], -1)


def oracle_vit(prm, img, heads, layers, theta, qk_norm):
    """taps [B, T, E] of the patch tokens in 64 bits from a dict of parameters"""
    x = F.conv2d(img.double(), prm['patch_embed.projection.weight'], prm['patch_embed.projection.bias'], stride=16)
    hw = x.shape[-2:]
    x = x.flatten(2).transpose(1, 2)
    x = torch.cat([prm['cls_token'].expand(x.shape[0], -1, -1), x], 1) + prm['pos_embed']
    B, N, E = x.shape
    taps = []
    for i in range(layers):
        q = lambda n: prm[f'layers.{i}.{n}']                                     # noqa: E731
        xn = F.layer_norm(x, (E,), q('ln1.weight'), q('ln1.bias'), EPS)
        qkv = xn @ q('attn.attn.in_proj_weight').t() + q('attn.attn.in_proj_bias')
        a, b, v = [t.reshape(B, N, heads, 64).transpose(1, 2) for t in qkv.split(E, -1)]
        if qk_norm:
            a, b = rms(a, q('attn.q_norm.weight')), rms(b, q('attn.k_norm.weight'))
        if theta:
            a, b = rotate(a, hw, theta), rotate(b, hw, theta)
        p = torch.softmax(torch.matmul(a, b.transpose(-1, -2)) / 8, -1)
        c = torch.matmul(p, v).transpose(1, 2).reshape(B, N, E)
        x = x + c @ q('attn.attn.out_proj.weight').t() + q('attn.attn.out_proj.bias')
        xn = F.layer_norm(x, (E,), q('ln2.weight'), q('ln2.bias'), EPS)
        hdn = F.gelu(xn @ q('ffn.layers.0.0.weight').t() + q('ffn.layers.0.0.bias'))
        x = x + hdn @ q('ffn.layers.1.weight').t() + q('ffn.layers.1.bias')
        taps.append(x[:, 1:])
    return taps


def close(got, ref, tol, what):
    got, ref = got.detach().double().cpu(), ref.detach().double()
    err = (got - ref).abs().max().item() / (ref.abs().max().item() + 1e-30)
    assert err <= tol, f'{what}: {err:.2e} of the largest magnitude > {tol:.0e}'


@pytest.mark.parametrize('qk_norm,theta', [(True, 100.0), (True, None), (False, 10.0)])
@pytest.mark.parametrize('img', [64, 96])
def test_vit_with_norm_and_rotation(qk_norm, theta, img):
    m = make_vit('fp32', img=img, qk_norm=qk_norm, rope_theta=theta)
    x = torch.randn(2, 3, img, img, generator=torch.Generator().manual_seed(5))
    prm = {n: p.detach().double().cpu().requires_grad_(True) for n, p in m.named_parameters()}
    ref = oracle_vit(prm, x, 4, 2, theta, qk_norm)
    outs = m(x.cuda())
    w = [torch.randn(t.shape, generator=torch.Generator().manual_seed(9 + i)) for i, t in enumerate(ref)]
    loss = sum((o.flatten(2).transpose(1, 2).double() * wi.double().cuda()).sum() for o, wi in zip(outs, w))
    loss.backward()
    sum((r * wi.double()).sum() for r, wi in zip(ref, w)).backward()
    torch.cuda.synchronize()
    for i, (o, r) in enumerate(zip(outs, ref)):
        close(o.flatten(2).transpose(1, 2), r, TOL['fp32'], f'tap {i}')
    for n, p in m.named_parameters():
        # the key bias has no gradient in exact arithmetic without the norm (a shift of all scores of a query): against in_proj as a whole
        close(p.grad, prm[n].grad, TOL['fp32'], n)


def saved_layers(loss_tensor):
    """the layers' autograd nodes behind a tensor"""
    seen, todo, out = set(), [loss_tensor.grad_fn], []
    while todo:
        f = todo.pop()
        if f is None or f in seen:
            continue
        seen.add(f)
        if type(f).__name__ == 'LayerFnBackward':
            out.append(f)
        todo += [g for g, _ in f.next_functions]
    return out


def back(t):
    """a saved activation as fp64 on the CPU, from its codes alone where it is a checkpoint"""
    from s4former_amd.functional import Packed
    if isinstance(t, Packed):
        s = torch.exp2(t.scales.cpu().double() - 127)
        return (t.codes.cpu().double().reshape(*s.shape, 32) * s[..., None]).reshape(t.shape)
    return t.detach().cpu().double()


def layer_backward(sv, prm, g2, B, N, E, H, qk_norm, tabs):
    """64-bit backward of one layer from what the product saved"""
    M = B * N
    f = lambda n: prm[n].detach().double().cpu()                                 # noqa: E731
    z = (sv['z'].cpu().double() - 25) / 192 if not hasattr(sv['z'], 'codes') and sv['z'].dtype == torch.uint8 else back(sv['z'])
    a, xn2, x1, ctx, qkv, xn, x = [back(sv[k]) for k in ('a', 'xn2', 'x1', 'ctxv', 'qkv', 'xn', 'x')]
    g = {}

    def ln(dy, xx, mean, rstd, gamma, name):
        mean, rstd = sv[mean].cpu().double()[:, None], sv[rstd].cpu().double()[:, None]
        xh = (xx.reshape(M, E) - mean) * rstd
        g[name + '.weight'], g[name + '.bias'] = (dy * xh).sum(0), dy.sum(0)
        w = dy * gamma
        return rstd * (w - w.mean(-1, keepdim=True) - xh * (w * xh).mean(-1, keepdim=True))
    g2 = g2.reshape(M, E)
    dz = (g2 @ f('ffn.layers.1.weight')) * z
    g['ffn.layers.1.weight'], g['ffn.layers.1.bias'] = g2.t() @ a, g2.sum(0)
    g['ffn.layers.0.0.weight'], g['ffn.layers.0.0.bias'] = dz.t() @ xn2, dz.sum(0)
    g1 = ln(dz @ f('ffn.layers.0.0.weight'), x1, 'mean2', 'rstd2', f('ln2.weight'), 'ln2') + g2
    g['attn.attn.out_proj.weight'], g['attn.attn.out_proj.bias'] = g1.t() @ ctx, g1.sum(0)
    dctx = g1 @ f('attn.attn.out_proj.weight')
    heads = lambda t: t.reshape(B, N, H, 64).transpose(1, 2)                     # noqa: E731
    q, k, v = [heads(t) for t in qkv.reshape(M, 3 * E).split(E, -1)]
    p = torch.exp(torch.matmul(q, k.transpose(-1, -2)) / 8 - sv['lse'].cpu().double()[..., None])
    dc = heads(dctx)
    ds = p * (torch.matmul(dc, v.transpose(-1, -2)) - (dc * heads(ctx)).sum(-1, keepdim=True))
    dq, dk, dv = torch.matmul(ds, k) / 8, torch.matmul(ds.transpose(-1, -2), q) / 8, torch.matmul(p.transpose(-1, -2), dc)
    if tabs is not None:
        turn = torch.complex(*[t.cpu().double() for t in tabs]).conj()
        dq, dk = [torch.cat([zz.real, zz.imag], -1) for zz in (torch.complex(t[..., :32], t[..., 32:]) * turn for t in (dq, dk))]
    if qk_norm:
        if isinstance(sv['pre'], tuple):
            s = torch.exp2(sv['pre'][1].cpu().double() - 127)
            pre = (sv['pre'][0].cpu().double().reshape(M, -1, 32) * s[..., None]).reshape(M, 2 * E)
        else:
            pre = sv['pre'].cpu().double()
        res = []
        for dy, xx, name in ((dq, pre[:, :E], 'attn.q_norm.weight'), (dk, pre[:, E:], 'attn.k_norm.weight')):
            xx = heads(xx)
            r = 1 / torch.sqrt((xx * xx).mean(-1, keepdim=True) + EPS)
            u = xx * r
            g[name] = (dy * u).sum((0, 1, 2))
            w = dy * f(name)
            res.append(r * (w - u * (w * u).mean(-1, keepdim=True)))
        dq, dk = res
    dqkv = torch.cat([t.transpose(1, 2).reshape(M, E) for t in (dq, dk, dv)], -1)
    g['attn.attn.in_proj_weight'], g['attn.attn.in_proj_bias'] = dqkv.t() @ xn, dqkv.sum(0)
    dx = ln(dqkv @ f('attn.attn.in_proj_weight'), x, 'mean1', 'rstd1', f('ln1.weight'), 'ln1') + g1
    return g, dx.reshape(B, N, E)


@pytest.fixture
def residual(request):
    from s4former_amd import runtime
    before = runtime._resid_fp32
    runtime.set_residual_fp32(request.param == 'fp32')
    yield request.param
    runtime.set_residual_fp32(before)


@pytest.mark.parametrize('dtype,residual', [('fp32', 'fp32'), ('bf16', 'fp32'), ('bf16', 'bf16')], indirect=['residual'])
@pytest.mark.parametrize('qk_norm,theta', [(True, 100.0), (False, None), (False, 100.0)])
def test_backward_from_checkpoints(dtype, residual, qk_norm, theta):
    """one layer: its gradients are the formulas' on the activations as the checkpoints restore them"""
    m = make_vit(dtype, layers=1, img=64, qk_norm=qk_norm, rope_theta=theta, act_q8=True)
    x = torch.randn(3, 3, 64, 64, generator=torch.Generator().manual_seed(5)).cuda()
    out = m(x)[0]
    (node,) = saved_layers(out)
    sv = dict(node.sv)
    assert hasattr(sv['a'], 'codes') and hasattr(sv['x'], 'codes') and sv['x'].dtype == (torch.bfloat16 if residual == 'bf16' else torch.float32)
    assert isinstance(sv['pre'], tuple) == qk_norm
    B, N, E = 3, 17, 256
    go = torch.randn(out.shape, generator=torch.Generator().manual_seed(8)).to(out.dtype).cuda()
    g2 = torch.zeros(B, N, E, dtype=torch.float64)
    g2[:, 1:] = go.detach().cpu().double().flatten(2).transpose(1, 2)
    prm = dict(m.layers[0].named_parameters())
    if dtype == 'bf16':
        prm = {n: (p.detach().bfloat16().float() if p.dim() == 2 else p) for n, p in prm.items()}
    ref, _ = layer_backward(sv, prm, g2, B, N, E, 4, qk_norm, m._rope((4, 4), x.device))
    out.backward(go)
    torch.cuda.synchronize()
    got = dict(m.layers[0].named_parameters())
    for n, r in ref.items():
        close(got[n].grad, r, TOL[dtype], n)


@pytest.mark.parametrize('dtype,residual', [('fp32', 'fp32'), ('bf16', 'fp32'), ('bf16', 'bf16')], indirect=['residual'])
@pytest.mark.parametrize('theta', [100.0, None])
def test_norm_backward_without_checkpoints(dtype, residual, theta):
    """one layer with qk_norm alone: queries and keys in front of the norm are kept in their own type and tensor; the gradients are the
    formulas' on what was kept"""
    m = make_vit(dtype, layers=1, img=64, qk_norm=True, rope_theta=theta)
    x = torch.randn(3, 3, 64, 64, generator=torch.Generator().manual_seed(5)).cuda()
    out = m(x)[0]
    (node,) = saved_layers(out)
    sv = dict(node.sv)
    B, N, E = 3, 17, 256
    assert torch.is_tensor(sv['pre']) and sv['pre'].shape == (B * N, 2 * E) and torch.is_tensor(sv['a'])
    go = torch.randn(out.shape, generator=torch.Generator().manual_seed(8)).to(out.dtype).cuda()
    g2 = torch.zeros(B, N, E, dtype=torch.float64)
    g2[:, 1:] = go.detach().cpu().double().flatten(2).transpose(1, 2)
    prm = dict(m.layers[0].named_parameters())
    if dtype == 'bf16':
        prm = {n: (p.detach().bfloat16().float() if p.dim() == 2 else p) for n, p in prm.items()}
    ref, _ = layer_backward(sv, prm, g2, B, N, E, 4, True, m._rope((4, 4), x.device))
    out.backward(go)
    torch.cuda.synchronize()
    got = dict(m.layers[0].named_parameters())
    assert set(ref) == set(got)
    for n, r in ref.items():
        close(got[n].grad, r, TOL[dtype], n)


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
def test_forward_is_untouched_and_less_is_kept(dtype):
    x = torch.randn(2, 3, 96, 96, generator=torch.Generator().manual_seed(5)).cuda()
    kept, outs = [], []
    for q8 in (False, True):
        m = make_vit(dtype, img=96, qk_norm=True, rope_theta=100.0, act_q8=q8)
        out = m(x)
        outs.append([o.detach().clone() for o in out])
        tensors = {}
        for node in saved_layers(out[-1]):
            for t in node.sv.values():
                for u in (t if isinstance(t, tuple) else (t.codes, t.scales) if hasattr(t, 'codes') else (t,)):
                    if torch.is_tensor(u):
                        tensors[u.data_ptr()] = u.numel() * u.element_size()
        kept.append(sum(tensors.values()))
        with torch.no_grad():
            again = m(x)
        assert all(torch.equal(a, b) for a, b in zip(out, again))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert kept[1] < (0.62 if dtype == 'bf16' else 0.45) * kept[0], kept


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
def test_options_in_the_training_step(dtype):
    """student, teacher, EMA and optimizer with all options on: two steps run, the gains move and the teacher follows them"""
    S.set_compute_dtype(dtype)
    cfg = C.tiny_model_cfg(unsup_weight=1.0, attn_mask_seperate_head=True, attn_mask_weight=5, adaptive_attn_mask=True)
    for k in ('backbone', 'backbone_ema'):
        cfg[k].update(qk_norm=True, rope_theta=100.0, act_q8=True)
    model = S.build_segmentor(cfg)
    model.train()
    C.load_filled(model, 1999, 60.0)
    model.cuda()
    opt = S.build_optimizer(model, dict(OPT))
    names = [n for n, _ in model.named_parameters() if n.endswith('q_norm.weight') or n.endswith('k_norm.weight')]
    assert len(names) == 2 * 2 * 4
    start = {n: p.detach().clone() for n, p in model.named_parameters() if n in names}
    for it in range(2):
        imgs, gt, metas = C.make_batch(2024 + it, 2, 2)
        opt.zero_grad()
        C.seed_host_rng(2024 + it)
        out = model.train_step(dict(img=imgs.cuda(), img_metas=metas, gt_semantic_seg=gt.cuda()), opt, iter=it)
        out['loss'].backward()
        torch.cuda.synchronize()
        grads = {n: p.grad.clone() for n, p in model.named_parameters() if n in names and p.requires_grad}
        assert grads and all(bool(torch.isfinite(g).all()) and float(g.abs().max()) > 0 for g in grads.values())
        opt.step()
    torch.cuda.synchronize()
    now = dict(model.named_parameters())
    for n in names:
        if n.startswith('backbone.'):
            assert not torch.equal(now[n], start[n]), n


@pytest.mark.parametrize('dtype', ['fp32', 'bf16'])
def test_teacher_gains_are_the_moving_average(dtype):
    """every step in front of the teacher's pass: gain <- m gain + (1 - m) the student's gain, for each of the teacher's gains.  m and 1 - m,
    the product and the sum are rounded once each: 4 half steps of the magnitudes"""
    S.set_compute_dtype(dtype)
    cfg = C.tiny_model_cfg(unsup_weight=1.0, attn_mask_seperate_head=True, attn_mask_weight=5, adaptive_attn_mask=True)
    for k in ('backbone', 'backbone_ema'):
        cfg[k].update(qk_norm=True, rope_theta=100.0, act_q8=True)
    model = S.build_segmentor(cfg)
    model.train()
    C.load_filled(model, 1999, 60.0)
    model.cuda()
    opt = S.build_optimizer(model, dict(OPT))
    gains = [n for n, _ in model.named_parameters() if n.startswith('backbone.') and n.endswith(('q_norm.weight', 'k_norm.weight'))]
    assert len(gains) == 2 * 4
    m = model.momentum_backbone
    assert 0 < m < 1

    def values(prefix):
        now = dict(model.named_parameters())
        return {n: now[n.replace('backbone.', prefix, 1)].detach().double().cpu().clone() for n in gains}
    for it in range(3):
        imgs, gt, metas = C.make_batch(2024 + it, 2, 2)
        student, teacher = values('backbone.'), values('backbone_ema.')
        opt.zero_grad()
        C.seed_host_rng(2024 + it)
        out = model.train_step(dict(img=imgs.cuda(), img_metas=metas, gt_semantic_seg=gt.cuda()), opt, iter=it)
        torch.cuda.synchronize()
        after = values('backbone_ema.')
        for n in gains:
            want, mag = m * teacher[n] + (1 - m) * student[n], m * teacher[n].abs() + (1 - m) * student[n].abs()
            assert bool(((after[n] - want).abs() <= 4 * 2.0 ** -24 * mag).all()), (it, n)
            moved = (1 - m) * (student[n] - teacher[n])
            assert float(moved.abs().max()) > 16 * 2.0 ** -24 * float(mag.max()), 'the values are too close for a skipped update to show'
        out['loss'].backward()
        opt.step()
        torch.cuda.synchronize()


@pytest.mark.parametrize('how', ['no_grad', 'inference_mode', 'frozen'])
@pytest.mark.parametrize('qk_norm', [False, True])
def test_nothing_is_kept_without_a_backward(monkeypatch, qk_norm, how):
    """a pass that no backward follows (teacher, inference, frozen parameters): nothing is packed or put aside; with act_q8 alone the layer is
    the plain one, with its one call a layer"""
    from s4former_amd import functional as Fn
    m = make_vit('fp32', qk_norm=qk_norm, act_q8=True)
    x = torch.randn(2, 3, 64, 64, generator=torch.Generator().manual_seed(5)).cuda()
    ref = [o.detach().clone() for o in m(x)]
    names, in_place = [], []
    call, norm = Fn.L.call, Fn.K.qk_norm_rope_fwd

    def spy_norm(a, b, *args, packed=None, **kw):
        in_place.append(a is b and packed is None)
        return norm(a, b, *args, packed=packed, **kw)
    monkeypatch.setattr(Fn.L, 'call', lambda name, *a, **k: (names.append(name), call(name, *a, **k))[1])
    monkeypatch.setattr(Fn.K, 'act_pack', lambda *a: names.append('act_pack'))
    monkeypatch.setattr(Fn.K, 'qk_norm_rope_fwd', spy_norm)
    if how == 'frozen':
        for p in m.parameters():
            p.requires_grad_(False)
        out = m(x)
    else:
        with getattr(torch, how)():
            out = m(x)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, ref))
    assert 'act_pack' not in names
    if qk_norm:
        assert in_place == [True, True]
    else:
        assert names.count('s4f_encoder_layer_fwd') == 2


def test_second_backward_is_refused():
    m = make_vit('fp32', layers=1, act_q8=True)
    out = m(torch.zeros(1, 3, 64, 64, device='cuda'))[0]
    out.sum().backward(retain_graph=True)
    with pytest.raises(S.S4FError, match='second time'):
        out.sum().backward()
