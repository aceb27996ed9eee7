"""Refusals of the query / key norm and of the 8-bit checkpoints, without a GPU: the typed front's, and the C entry points' (which check
before anything is launched)."""
import pytest
import torch

from s4former_amd import _lib as L
from s4former_amd import kernels as K
from s4former_amd._lib import S4FError

P = 1 << 20            # stands for an aligned device address: refused calls never read it


def refused(name, args, match):
    lib = L.load()
    assert getattr(lib, name)(*args) != 0
    msg = lib.s4f_last_error().decode()
    assert match in msg, msg


FWD = dict(x=P, ldx=128, y=P, ldy=128, gq=P, gk=P, cos=P, sin=P, period=4, eps=1e-6, codes=None, scales=None, rows=8, Hq=1, Hk=1, dtype=1, stream=None)
BWD = dict(dy=P, lddy=128, x=P, ldx=128, codes=None, scales=None, dx=P, lddx=128, gq=P, gk=P, cos=P, sin=P, period=4, eps=1e-6, dgq=P, dgk=P,
           accumulate=0, ws=P, ws_bytes=1 << 20, rows=8, Hq=1, Hk=1, dtype=1, stream=None)


@pytest.mark.parametrize('change,match', [
    (dict(dtype=2), 'dtype'), (dict(rows=0), 'positive'), (dict(Hq=0), 'positive'), (dict(Hk=-1), 'positive'),
    (dict(rows=1 << 31, period=1 << 31), '2^31'), (dict(gk=None), 'pairs'), (dict(sin=None), 'pairs'),
    (dict(gq=None, gk=None, cos=None, sin=None), 'neither'), (dict(eps=0.0), 'eps'), (dict(eps=float('nan')), 'eps'), (dict(eps=float('inf')), 'eps'),
    (dict(eps=1e-39), 'eps'), (dict(rows=1 << 61, period=4, Hq=4, Hk=4, ldx=512, ldy=512), '2^31'), (dict(rows=1 << 29), 'one launch'),
    (dict(rows=(1 << 28), dtype=0), 'one launch'),
    (dict(period=3), 'divide'), (dict(period=0), 'divide'), (dict(period=16), 'divide'), (dict(x=None), 'null'), (dict(y=None), 'null'),
    (dict(x=P + 2), '16-byte'), (dict(ldx=129), '16-byte'), (dict(ldy=130), '16-byte'), (dict(ldy=120), 'overlap'), (dict(gq=P + 4), 'aligned'),
    (dict(cos=P + 8), 'aligned'), (dict(codes=P), 'checkpoint'), (dict(scales=P), 'checkpoint'), (dict(codes=P + 8, scales=P), 'alignment'),
    (dict(codes=P, scales=P + 1), 'alignment'), (dict(gq=None, gk=None, codes=P, scales=P), 'checkpoint'),
])
def test_forward_entry_refuses(change, match):
    refused('s4f_qk_norm_rope_fwd', {**FWD, **change}.values(), match)


@pytest.mark.parametrize('change,match', [
    (dict(dtype=-1), 'dtype'), (dict(rows=-5), 'positive'), (dict(gq=None), 'pairs'), (dict(period=5), 'divide'), (dict(dy=None), 'null'),
    (dict(dx=P + 8), '16-byte'), (dict(lddx=64), 'overlap'), (dict(x=None), 'not both'), (dict(codes=P, scales=P), 'not both'),
    (dict(x=None, codes=P), 'not both'), (dict(ldx=-128), '16-byte'), (dict(dgq=None), 'workspace'), (dict(ws=None), 'workspace'),
    (dict(ws=P + 4), 'workspace'), (dict(ws_bytes=8), 'too small'),
])
def test_backward_entry_refuses(change, match):
    refused('s4f_qk_norm_rope_bwd', {**BWD, **change}.values(), match)


PACK = dict(x=P, ldx=64, codes=P, scales=P, rows=4, C=64, dtype=1, stream=None)


@pytest.mark.parametrize('change,match', [
    (dict(dtype=7), 'dtype'), (dict(x=None), 'null'), (dict(codes=None), 'null'), (dict(scales=None), 'null'), (dict(rows=0), 'positive'),
    (dict(C=0), '32'), (dict(C=48), '32'), (dict(C=-32), '32'), (dict(x=P + 2), '16-byte'), (dict(ldx=68), '16-byte'), (dict(ldx=-64), '16-byte'),
    (dict(codes=P + 4), '16-byte'), (dict(rows=1 << 50), 'too large'), (dict(rows=1 << 31), 'too large'), (dict(ldx=128, rows=1 << 31), 'too large'),
])
def test_pack_entries_refuse(change, match):
    a = {**PACK, **change}
    refused('s4f_act_pack', a.values(), match)
    refused('s4f_act_unpack', (a['codes'], a['scales'], a['x'], a['ldx'], a['rows'], a['C'], a['dtype'], None), match)


def test_unpack_entry_refuses_overlapping_rows():
    refused('s4f_act_unpack', (P, P, P, 32, 4, 64, 1, None), 'overlap')


WG = dict(dy=P, lddy=64, codes=P, scales=P, out=P, rows=4096, M=64, N=64)


@pytest.mark.parametrize('change,match', [
    (dict(dy=None), 'null'), (dict(codes=None), 'null'), (dict(scales=None), 'null'), (dict(out=None), 'null'), (dict(M=12), 'multiple'),
    (dict(N=40), 'multiple'), (dict(M=0), 'multiple'), (dict(rows=0), 'multiple'), (dict(lddy=68), '16-byte'), (dict(dy=P + 8), '16-byte'),
    (dict(out=P + 4), '16-byte'), (dict(lddy=0), 'overlap'), (dict(lddy=-64), 'overlap'), (dict(lddy=56), 'overlap'), (dict(lddy=1 << 23), 'too large'),
    (dict(lddy=1 << 22), 'too large'), (dict(N=1 << 23), 'too large'),
    (dict(N=1 << 24), 'too large'), (dict(rows=(1 << 31) - 100), 'too large'), (dict(rows=1 << 40), 'too large'), (dict(M=1 << 20, N=1 << 20, lddy=1 << 20), 'too large'), (dict(), 'workspace'),
])
def test_wgrad_entry_refuses(change, match):
    good, bad = L.WgradPackedDesc(**WG), L.WgradPackedDesc(**{**WG, **change})
    arr = (L.WgradPackedDesc * 2)(good, bad)
    refused('s4f_wgrad_packed', (arr, 2, 1, 0, None, 0, None), match)


def test_wgrad_entry_refuses_counts():
    arr = (L.WgradPackedDesc * 5)(*[L.WgradPackedDesc(**WG)] * 5)
    for n in (0, 5, -1):
        refused('s4f_wgrad_packed', (arr, n, 1, 0, P, 1 << 30, None), 'problems')
    refused('s4f_wgrad_packed', (None, 1, 1, 0, P, 1 << 30, None), 'problems')
    refused('s4f_wgrad_packed', (arr, 1, 3, 0, P, 1 << 30, None), 'dtype')


def test_workspace_queries():
    assert K.qk_norm_rope_ws_bytes(0, 1, 1) == 0 and K.wgrad_packed_ws_bytes([(8, 32, 0)], 1) == 0
    one = K.qk_norm_rope_ws_bytes(1, 1, 1)
    assert 0 < one <= K.qk_norm_rope_ws_bytes(1000, 12, 12) <= K.qk_norm_rope_ws_bytes(1 << 20, 16, 16)
    assert K.wgrad_packed_ws_bytes([(8, 32, 1)], 1) == 0                          # one range of rows: no slabs
    for bad in ([(12, 32, 5)], [(8, 33, 5)], [(8, 32, -1)], [(8, 32, 5)] * 5):
        with pytest.raises(S4FError):
            K.wgrad_packed_ws_bytes(bad, 1)
    with pytest.raises(S4FError):
        K.workspace_bytes(K.WS_QK_NORM, 4, 0, 1)
    for bad in ((1 << 61, 4, 4), (4, (5 - (1 << 32)), 1), (4, 1, 1 << 32)):
        with pytest.raises(S4FError):
            K.workspace_bytes(K.WS_QK_NORM, *bad)
    with pytest.raises(S4FError):
        K.wgrad_packed_ws_bytes([(8 - (1 << 32), 32, 5)], 1)


def test_front_refuses():
    """what the typed front says before a pointer is taken: shapes, types, host tensors"""
    z = torch.zeros
    i8, u8, g = lambda *s: z(*s, dtype=torch.int8), lambda *s: z(*s, dtype=torch.uint8), z(64)          # noqa: E731
    for call in (
        lambda: K.act_pack(z(4, 64), i8(4, 64), u8(4, 2), 0),                                            # host tensors
        lambda: K.act_pack(z(4, 48), i8(4, 48), u8(4, 1), 0),
        lambda: K.act_pack(z(4, 64), i8(4, 64), u8(4, 2), 1),                                            # fp32 tensor, bf16 asked
        lambda: K.act_pack(z(4, 2, 32), i8(4, 64), u8(4, 2), 0),
        lambda: K.act_unpack(i8(4, 64), u8(4, 2), z(4, 0), 0),
        lambda: K.qk_norm_rope_fwd(z(4, 128), z(4, 128), 1, 1, 0, gq=g, gk=g),
        lambda: K.qk_norm_rope_fwd(z(4, 192), z(4, 128), 1, 1, 0, gq=g, gk=g),
        lambda: K.qk_norm_rope_bwd(z(4, 128), z(4, 128), 1, 1, 0, x=z(4, 128), gq=g, gk=g, dgq=g, dgk=g),
        lambda: K.wgrad_packed([], 0),
        lambda: K.wgrad_packed([(z(4, 8), i8(4, 32), u8(4, 1), z(8, 33))], 0),
        lambda: K.wgrad_packed([(z(4, 8), i8(4, 32), u8(4, 1), z(8, 32))], 0),
        lambda: K.wgrad_packed([(z(4, 8), i8(4, 32), u8(4, 1), z(8, 32))] * 5, 0),
    ):
        with pytest.raises(S4FError):
            call()


FAR = 1 << 30          # apart from P by more than any of these tensors


@pytest.mark.parametrize('change', [dict(codes=P + 512, scales=P + 2 * FAR), dict(codes=P + FAR, scales=P + 2046), dict(codes=P + FAR, scales=P + FAR + 1022),
                                    dict(y=P + 3 * FAR, codes=P + 3 * FAR + 2032, scales=P + FAR)])
def test_forward_entry_refuses_overlap(change):
    # x and y: 8 rows of 256 bytes
    refused('s4f_qk_norm_rope_fwd', {**FWD, **change}.values(), 'overlaps')


# rows of 256 bytes: one element, half a row, a row on, other strides over the same memory, slices of one buffer that share columns
MEET = [dict(y=P + 16), dict(y=P + 128), dict(y=P + 256), dict(y=P - 256), dict(ldx=384, ldy=384, y=P + 240), dict(ldx=384, ldy=384, y=P + 528),
        dict(ldx=384, ldy=256), dict(ldx=0), dict(ldy=256), dict(ldx=192, ldy=192, y=P + 128)]


@pytest.mark.parametrize('change', MEET)
def test_rows_that_meet_are_refused(change):
    refused('s4f_qk_norm_rope_fwd', {**FWD, **change}.values(), 'x and y overlap')
    to = dict(x='dy', y='dx', ldx='lddy', ldy='lddx')
    back = {to[k]: v for k, v in change.items()}
    refused('s4f_qk_norm_rope_bwd', {**BWD, **dict(x=P + 2 * FAR, ws=P + 4 * FAR, dgq=P + 5 * FAR, dgk=P + 6 * FAR), **back}.values(), 'dy and dx overlap')
    to = dict(x='x', y='dx', ldx='ldx', ldy='lddx')
    back = {to[k]: v for k, v in change.items()}
    refused('s4f_qk_norm_rope_bwd', {**BWD, **dict(dy=P + 2 * FAR, ws=P + 4 * FAR, dgq=P + 5 * FAR, dgk=P + 6 * FAR), **back}.values(), 'x and dx overlap')


@pytest.mark.parametrize('change', [dict(dgk=P + 5 * FAR + 252), dict(ws=P + FAR + 2032), dict(ws=P + 5 * FAR), dict(ws=P + 2 * FAR + 16), dict(dgq=P + FAR),
                                    dict(x=None, codes=P + FAR + 16, scales=P + 8 * FAR), dict(x=None, codes=P + 8 * FAR, scales=P + FAR + 2046)])
def test_backward_entry_refuses_overlap(change):
    apart = dict(dy=P, x=P + 2 * FAR, dx=P + FAR, ws=P + 4 * FAR, dgq=P + 5 * FAR, dgk=P + 6 * FAR)
    refused('s4f_qk_norm_rope_bwd', {**BWD, **apart, **change}.values(), 'overlap')


@pytest.mark.parametrize('codes,scales', [(P + 512 - 16, P + FAR), (P - 256 + 16, P + FAR), (P + FAR, P + 511), (P + FAR, P + FAR + 255), (P, P + FAR)])
def test_pack_entries_refuse_overlap(codes, scales):
    # 4 rows of 64 bf16 values: 512 bytes, codes 256, scales 8
    refused('s4f_act_pack', (P, 64, codes, scales, 4, 64, 1, None), 'overlap')
    refused('s4f_act_unpack', (codes, scales, P, 64, 4, 64, 1, None), 'overlap')


@pytest.mark.parametrize('second', [dict(out=P + 16), dict(dy=P + 4 * 64 * 64 - 16), dict(codes=P), dict(scales=P + 5), dict(dy=P + 9 * FAR + 16), dict(scales=P + 9 * FAR)])
def test_wgrad_entry_refuses_overlap(second):
    far = dict(dy=P + 2 * FAR, codes=P + 3 * FAR, scales=P + 4 * FAR, out=P + 5 * FAR, rows=16400)
    first = dict(WG, dy=P + 6 * FAR, codes=P + 7 * FAR, scales=P + 8 * FAR, out=P, rows=16400)
    arr = (L.WgradPackedDesc * 2)(L.WgradPackedDesc(**first), L.WgradPackedDesc(**{**WG, **far, **second}))
    refused('s4f_wgrad_packed', (arr, 2, 1, 0, P + 9 * FAR, 1 << 28, None), 'overlap')


def test_rows_apart_pass_the_overlap_check():
    # the same matrix, one behind the other, column slices of one buffer, a broadcast row in front of the output: the next check refuses
    for change in (dict(), dict(y=P + 2048), dict(y=P - 2048), dict(ldx=384, ldy=384, y=P + 256), dict(ldx=384, ldy=384, y=P + 512), dict(ldx=0, y=P + 256)):
        refused('s4f_qk_norm_rope_fwd', {**FWD, **change, 'codes': P + FAR, 'scales': P + FAR}.values(), 'checkpoint overlaps')


# 8 rows of 256 bytes; gains of 256 bytes; tables of 4 positions, 512 bytes
PAR = dict(gq=P + 9 * FAR, gk=P + 9 * FAR + 256, cos=P + 10 * FAR, sin=P + 10 * FAR + 512)
ONTO = [('gq', 240), ('gk', 240), ('cos', 496), ('sin', 496), ('gq', 0), ('cos', 0)]


@pytest.mark.parametrize('of,off', ONTO)
def test_forward_refuses_writes_to_gains_and_tables(of, off):
    at = PAR[of] + off
    for change in (dict(y=at), dict(codes=at, scales=P + 3 * FAR), dict(codes=P + 3 * FAR, scales=at), dict(y=at - 2048 + 16)):
        refused('s4f_qk_norm_rope_fwd', {**FWD, **PAR, 'y': P + 2 * FAR, **change}.values(), 'gains or the tables')
    if of in ('cos', 'sin'):                                 # the rotation alone
        refused('s4f_qk_norm_rope_fwd', {**FWD, **PAR, 'gq': None, 'gk': None, 'y': at}.values(), 'gains or the tables')


@pytest.mark.parametrize('of,off', ONTO)
def test_backward_refuses_writes_to_gains_and_tables(of, off):
    at = PAR[of] + off
    apart = {**BWD, **PAR, **dict(dy=P, x=P + 2 * FAR, dx=P + FAR, ws=P + 4 * FAR, dgq=P + 5 * FAR, dgk=P + 6 * FAR)}
    for change in (dict(dx=at), dict(ws=at), dict(dgq=at), dict(dgk=at), dict(ws=at - (1 << 20) + 16)):
        refused('s4f_qk_norm_rope_bwd', {**apart, **change}.values(), 'gains or the tables')
    if of in ('cos', 'sin'):
        refused('s4f_qk_norm_rope_bwd', {**apart, 'gq': None, 'gk': None, 'dx': at}.values(), 'gains or the tables')


@pytest.mark.parametrize('change', [dict(dgq=P + 2032), dict(dgk=P + 2 * FAR), dict(x=None, codes=P + 7 * FAR, scales=P + 8 * FAR, dgq=P + 7 * FAR + 512),
                                    dict(x=None, codes=P + 7 * FAR, scales=P + 8 * FAR, dgk=P + 8 * FAR + 16)])
def test_backward_refuses_gain_gradients_over_inputs(change):
    apart = {**BWD, **PAR, **dict(dy=P, x=P + 2 * FAR, dx=P + FAR, ws=P + 4 * FAR, dgq=P + 5 * FAR, dgk=P + 6 * FAR)}
    refused('s4f_qk_norm_rope_bwd', {**apart, **change}.values(), 'overlap')


@pytest.mark.parametrize('dtype', [-1, 2, 1 << 32])
def test_workspace_query_refuses_types(dtype):
    with pytest.raises(S4FError):
        K.workspace_bytes(K.WS_WGRAD_PACKED, dtype, 64, 64, 4096)


# ------------------------------------------------------------------------------------------------------------- options of the backbone
def test_backbone_options():
    import s4former_amd as S
    from tests import common as C
    plain = C.tiny_model_cfg(unsup_weight=1.0)
    keys = set(S.build_segmentor(plain).state_dict())
    cfg = C.tiny_model_cfg(unsup_weight=1.0)
    for k in ('backbone', 'backbone_ema'):
        cfg[k].update(qk_norm=True, rope_theta=100.0, act_q8=True)
    m = S.build_segmentor(cfg)
    more = set(m.state_dict()) - keys
    assert keys <= set(m.state_dict())
    assert more == {f'{b}.layers.{i}.attn.{n}_norm.weight' for b in ('backbone', 'backbone_ema') for i in range(4) for n in 'qk'}
    assert all(tuple(m.state_dict()[k].shape) == (64,) and bool((m.state_dict()[k] == 1).all()) for k in more)
    m._build_stores()
    for bad in (0.0, -1.0, 0.5, float('inf'), float('nan')):
        cfg['backbone']['rope_theta'] = bad
        with pytest.raises(S4FError):
            S.build_segmentor(cfg)
    cfg['backbone']['rope_theta'] = 10.0
    with pytest.raises(S4FError, match='rope_theta'):
        S.build_segmentor(cfg)._build_stores()
    cfg['backbone']['rope_theta'] = 100.0
    cfg['backbone_ema']['qk_norm'] = False
    with pytest.raises(S4FError, match='line up'):
        S.build_segmentor(cfg)._build_stores()


def test_axial_tables():
    from s4former_amd.vit import axial_rope_tables
    cos, sin = axial_rope_tables(3, 5, 100.0, 'cpu')
    assert cos.shape == sin.shape == (16, 32) and cos.dtype == torch.float32
    assert bool((cos[0] == 1).all()) and bool((sin[0] == 0).all())                # the cls token is not turned
    row, col, i = 2, 4, 5
    t = 1 + row * 5 + col
    a, b = torch.tensor(row * 100.0 ** (-i / 16), dtype=torch.float64), torch.tensor(col * 100.0 ** (-i / 16), dtype=torch.float64)
    assert cos[t, i] == a.cos().float() and sin[t, i] == a.sin().float() and cos[t, 16 + i] == b.cos().float() and sin[t, 16 + i] == b.sin().float()


def test_rotation_tables_do_not_pile_up():
    from s4former_amd import vit
    m = vit.VisionTransformer(img_size=64, embed_dims=128, num_layers=1, num_heads=2, rope_theta=100.0)
    grids = [(h, w) for h in range(1, 13) for w in range(1, 13)]
    for hw in grids * 2:
        got, want = m._rope(hw, 'cpu'), vit.axial_rope_tables(*hw, 100.0, 'cpu')
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert len(m._rope_tables) == vit.ROPE_GRIDS < len(grids)
    assert m._rope(grids[0], 'cpu')[0] is m._rope(grids[0], 'cpu')[0]              # a kept one is the same each time
