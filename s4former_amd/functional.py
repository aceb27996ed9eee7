"""Coarse-grained autograd nodes of the hot path.  Each node is a fixed sequence of C-ABI kernel launches with a
hand-written backward; parameter gradients are accumulated by the kernels straight into the flat gradient
arena (ParamStore.grad) and the node returns None for them, so a step costs ~20 autograd nodes instead of
the reference's several hundred ATen ops per pass (SURVEY §7 "host overhead").

Reference semantics restated here:
  PatchEmbedFn   models/utils/embed.py:183-204 + vit.py:486-487,445 (cls concat, + pos_embed)
  LayerFn        vit.py:113-127 TransformerEncoderLayer (LN -> MHA -> +x ; LN -> FFN(GELU erf) -> +x)
  HeadLossFn     setr_up_head.py:92-111 + decode_head.py:318-355 + cross_entropy_loss.py:45-61 (mean over ALL
                 pixels, Q5).  conv_seg is applied before the last bilinear upsample (they commute: both
                 linear, interpolation weights sum to 1) and the upsample is fused into the CE kernels.
"""
import os

import torch
import torch.distributed as dist
from torch.autograd import Function

from . import kernels as K
from . import runtime
from . import _lib as L
from ._lib import BF16, F32, S4FError

SKIP_MASKED_COPY = os.environ.get('S4F_SKIP_MASKED_COPY', '1') != '0'     # A/B switch of head_backward's s = 1 stages
FUSE_CLS_FWD = os.environ.get('S4F_FUSE_CLS_FWD', '1') != '0'             # A/B switch: BN + ReLU + conv_seg forward in one pass
FUSE_CLS_WGRAD = os.environ.get('S4F_FUSE_CLS_WGRAD', '1') != '0'         # A/B switch: conv_seg weight gradient inside the BN statistics pass (no stored activation)
FUSE_CLS_GRAD = os.environ.get('S4F_FUSE_CLS_GRAD', '1') != '0'           # A/B switch: conv_seg input gradient inside the BN backward passes
# experiment (round 4): the LAST stage of an inference-only head pass (the teacher's pseudo-label path) with fp32
# operands inside a bf16 run - the last conv's output is kept in fp32 and BN + ReLU + conv_seg run on it with the fp32 master
# conv_seg weights.  Measured label flip rate against the reference: DESIGN A.15.  Off by default.
TEACHER_LAST_FP32 = os.environ.get('S4F_TEACHER_LAST_FP32', '0') != '0'
LOGIT_LD = 32   # channel stride of the low-resolution logits buffers (>= num_classes, multiple of 8)

# ---------------------------------------------------------------------------------------------- side stream
# Weight-gradient GEMMs and bias column sums do not feed the backward chain (they only accumulate into the gradient
# arena), so they are enqueued on a second HIP stream: they fill the CUs that the tail of each chain kernel leaves
# idle (tile-count quantisation: 768..1152 tiles over 256 CUs).  The optimiser / gradient reducer joins the stream.
USE_SIDE_STREAM = os.environ.get('S4F_SIDE_STREAM', '1') != '0'
# A/B switch (round 3): the grouped weight gradient of an encoder layer on the side stream (1) or inside the backward chain (0).
# A block of the 8-wave GEMMs holds a CU's whole register file (2 waves x 256 registers per SIMD): while the 216 blocks of the
# grouped weight gradient are resident, the chain's kernels run on the 40 CUs that are left.
LAYER_WG_SIDE = os.environ.get('S4F_LAYER_WG_SIDE', '1') != '0'
# A/B switch (round 4): the image groups of a backbone tap share one gradient buffer written by the heads (TapSplitFn) instead
# of autograd's slice / zero-fill / add plumbing
TAP_SPLIT = os.environ.get('S4F_TAP_SPLIT', '1') != '0'
_side = {}


def side_stream(device):
    key = torch.device(device).index
    if key not in _side:
        _side[key] = torch.cuda.Stream(device=device)
    return _side[key]


_head = {}                     # (device index, name) -> stream the decode / auxiliary heads run on
GRAD_CONSUMER = None           # stream that consumes the token gradients of a head launched on a head stream
USE_HEAD_STREAMS = os.environ.get('S4F_HEAD_STREAMS', '1') != '0'


def head_stream(device, name, priority=0):
    key = (torch.device(device).index, name)
    if key not in _head:
        _head[key] = torch.cuda.Stream(device=device, priority=priority)
    return _head[key]


_burn = []


def pretouch_streams(device, order, optimizer=None):
    """use the package's streams for the first time in a given order ('decode', 'aux', 'side', 'opt', 'burn' = a throw-away
    stream): the runtime binds a stream to one of its four hardware queues at its FIRST use, so the order decides which streams
    share a queue (two streams on one queue serialise)."""
    def touch(st):
        with torch.cuda.stream(st):
            torch.empty(64, device=device).fill_(0.0)
    for name in order:
        if name == 'burn':
            _burn.append(torch.cuda.Stream(device=device))
            touch(_burn[-1])
        elif name == 'side':
            touch(side_stream(device))
        elif name == 'opt':
            if optimizer is not None:
                if getattr(optimizer, '_stream', None) is None:
                    optimizer._stream = torch.cuda.Stream(device=device)
                touch(optimizer._stream)
        else:
            touch(head_stream(device, name))
    torch.cuda.synchronize(device)


def check_stream_layout(device, cycles=400_000, extra=()):
    """Do the chain's stream, the two head streams and the weight-gradient stream run CONCURRENTLY (= sit on different hardware
    queues)?  Two single-thread spin kernels (torch.cuda._sleep) started together on a pair of streams take about one spin if
    the streams are on different queues and two if they share one.  Returns dict(ok=bool, pairs={name: ratio}); ok = every
    pair overlapped (ratio < 1.5).  A few hundred microseconds, once, at set-up."""
    res = dict(ok=False, pairs={})
    try:
        names = [('main', torch.cuda.current_stream(device)), ('decode', head_stream(device, 'decode')), ('aux', head_stream(device, 'aux')),
                 ('side', side_stream(device))] + [(n, st) for n, st in extra if st is not None]

        def timed(streams):
            torch.cuda.synchronize(device)
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            cur = torch.cuda.current_stream(device)
            e0.record(cur)
            for st in streams:
                st.wait_event(e0) if st != cur else None
                with torch.cuda.stream(st):
                    torch.cuda._sleep(cycles)
            for st in streams:
                if st != cur:
                    cur.wait_stream(st)
            e1.record(cur)
            torch.cuda.synchronize(device)
            return e0.elapsed_time(e1)
        timed([names[0][1]])                                  # warm-up
        one = min(timed([names[0][1]]) for _ in range(3))
        # `ok` judges only the pairs the first-use order is MEANT to separate: the four compute streams among themselves and the
        # communication stream against the chain.  With more streams than the runtime has hardware queues (four) SOME pair shares a
        # queue by pigeonhole: the remaining pairs (comm / opt against the head and weight-gradient streams) are reported, not judged.
        core = {'main', 'decode', 'aux', 'side'}
        ok = True
        for i in range(len(names)):
            for j in range(i + 1, len(names)):
                t = min(timed([names[i][1], names[j][1]]) for _ in range(2))
                r = t / max(one, 1e-6)
                res['pairs'][f'{names[i][0]}+{names[j][0]}'] = round(r, 2)
                judged = ({names[i][0], names[j][0]} <= core) or ({names[i][0], names[j][0]} == {'main', 'comm'})
                if judged:
                    ok = ok and r < 1.5
                else:
                    res.setdefault('informational', []).append(f'{names[i][0]}+{names[j][0]}')
        res['ok'] = ok
    except Exception as e:                                    # noqa: BLE001 - a missing _sleep or an odd runtime: no claim, fall back
        res['error'] = f'{type(e).__name__}: {e}'
    return res


def extra_streams(device=None):
    """every stream besides the caller's that this package launches compute kernels on"""
    idx = None if device is None else torch.device(device).index
    return [st for st in list(_side.values()) + list(_head.values()) if idx is None or st.device.index == idx]


def join_side_streams():
    """make the current stream wait for everything enqueued on the side / head stream(s)"""
    cur = torch.cuda.current_stream()
    for st in extra_streams(cur.device):
        cur.wait_stream(st)


class on_head_stream:
    """with on_head_stream(dev, name): the head's forward (and therefore, by autograd's stream rule, its backward) runs on
    its own stream after everything enqueued so far.  The decode head and the auxiliary heads are independent given the
    backbone taps; their HBM-bound BN / upsample kernels then overlap the other head's conv GEMMs."""

    def __init__(self, device, name):
        self.dev, self.name = device, name
        self.on = USE_HEAD_STREAMS and torch.device(device).type == 'cuda'

    def __enter__(self):
        global GRAD_CONSUMER
        if not self.on:
            return self
        main = torch.cuda.current_stream()
        if any(main == st for st in _head.values()):
            self.on = False                       # already on a head stream (nested use): stay there
            return self
        self.st = head_stream(self.dev, self.name, main.priority)
        self.st.wait_stream(main)
        self.prev_consumer = GRAD_CONSUMER
        GRAD_CONSUMER = main
        self.ctx = torch.cuda.stream(self.st)
        self.ctx.__enter__()
        return self

    def __exit__(self, *exc):
        global GRAD_CONSUMER
        if not self.on:
            return False
        self.ctx.__exit__(*exc)
        GRAD_CONSUMER = self.prev_consumer
        return False


class on_side:
    """with on_side(dev, t1, t2, ...): kernels launched inside run on the side stream after everything already enqueued
    on the current stream; the tensors are kept alive for the side stream (caching-allocator record_stream)."""

    def __init__(self, device, *tensors, enable=True):
        self.dev, self.tensors = device, tensors
        self.enable = enable and USE_SIDE_STREAM

    def __enter__(self):
        if not self.enable:
            return self
        self.side = side_stream(self.dev)
        self.side.wait_stream(torch.cuda.current_stream())
        self.ctx = torch.cuda.stream(self.side)
        self.ctx.__enter__()
        return self

    def __exit__(self, *exc):
        if not self.enable:
            return False
        self.ctx.__exit__(*exc)
        for t in self.tensors:
            if t is not None:
                t.record_stream(self.side)
        return False


def _T(code):
    return torch.bfloat16 if code == BF16 else torch.float32


def _lp(t):
    """device pointer for a launch descriptor (None -> NULL)"""
    return None if t is None else t.data_ptr()


def _R(code):
    """torch dtype of the residual stream (token tensors between the layers and their gradients): fp32 in parity mode, the
    operand type in bf16 mode unless S4F_RESID=fp32 (runtime.residual_dtype)"""
    return torch.bfloat16 if (code == BF16 and runtime.residual_dtype() == BF16) else torch.float32


def _gemm_resid(A, W, M, N, Kd, code, bias, resid, out, **kw):
    """out[M, N] = A W^T + bias + resid, out / resid in the residual-stream type"""
    if out.dtype == torch.bfloat16:
        K.gemm(A, W, M, N, Kd, Kd, Kd, code, bias=bias, resid=resid, ldr=N if resid is not None else 0, out_t=out, ldo_t=N, **kw)
    else:
        K.gemm(A, W, M, N, Kd, Kd, Kd, code, bias=bias, resid=resid, ldr=N if resid is not None else 0, out_f32=out, ldo_f32=N, **kw)


class _ZeroPool:
    """The step needs ~60 small zero-initialised fp32 accumulators (BN sums, loss sums, column sums).  One buffer,
    re-zeroed with ONE kernel at the start of forward_train, hands out slices instead of ~60 fill launches.  A slice is
    valid until the next step begins; nothing that outlives the step may alias it."""
    ELEMS = 1 << 18

    def __init__(self):
        self.buf, self.off = None, 0

    def begin(self, device):
        device = torch.device(device)
        if self.buf is None or self.buf.device != device:
            self.buf = torch.zeros(self.ELEMS, device=device)
        elif self.off:
            self.buf[:self.off].zero_()
        self.off = 0

    def take(self, n, device):
        n_al = (n + 63) // 64 * 64
        if self.buf is None or self.buf.device != torch.device(device) or self.off + n_al > self.ELEMS:
            return torch.zeros(n, device=device)
        v = self.buf[self.off:self.off + n]
        self.off += n_al
        return v


ZERO_POOL = _ZeroPool()


def zeros_small(n, device):
    return ZERO_POOL.take(n, device)


def _splitk(tiles, nk, target=512):
    sk = max(1, target // max(1, tiles))
    return int(max(1, min(sk, max(1, nk // 4))))


def _tiles256(m, n):
    return ((m + 255) // 256) * ((n + 255) // 256)


def _tiles(m, n):
    return ((m + 127) // 128) * ((n + 127) // 128)


def _nk(k, code):
    bk = 64 if code == BF16 else 32
    return (k + bk - 1) // bk


def _as_T(x_f32, code):
    """operand-typed copy of an fp32 tensor (identity in parity mode)"""
    if code == F32:
        return x_f32
    cached = getattr(x_f32, '_s4f_t', None)
    if cached is not None and cached[1] == x_f32._version and cached[2] == x_f32.data_ptr():
        return cached[0]
    out = torch.empty(x_f32.shape, device=x_f32.device, dtype=torch.bfloat16)
    K.cast(x_f32, out, BF16)
    return out


def _handed_colsum(g):
    """column sums [E] of a gradient tensor if the node that produced it left them on it (LayerFn.backward), else None"""
    cached = getattr(g, '_s4f_colsum', None)
    if cached is not None and cached[1] == g._version and cached[2] == g.data_ptr():
        return cached[0]
    return None


def _dgrad(dy, w, M, N, Kd, store, code, **epi):
    """dx[M, N] = dy[M, Kd] W[Kd, N]  (W = F.linear weight [out = Kd, in = N]).  bf16: row-major x row-major against the
    transposed shadow W^T [N][Kd] (the fastest kernel forms, incl. the 8-wave ping-pong one); fp32: W read k-major.
    Returns True if a requested colsum= was folded into the launch."""
    if code == BF16:
        return K.gemm(dy, store.shadow_T(w), M, N, Kd, Kd, Kd, code, **epi)
    epi.pop('colsum', None)
    K.gemm(dy, store.shadow(w), M, N, Kd, Kd, N, code, b_mode=K.OP_K, **epi)
    return False


def _wgrad(dy, x, M, N, rows, ldm, ldn, out, code):
    """out[M,N] += dy[rows,M]^T x[rows,N]   (fp32 atomic accumulate into the gradient arena)"""
    K.gemm(dy, x, M, N, rows, ldm, ldn, code, a_mode=K.OP_K, b_mode=K.OP_K, out_f32=out, ldo_f32=N, atomic=True,
           splitk=_splitk(_tiles(M, N), _nk(rows, code)))


# ============================================================================================== patch embed
class PatchEmbedFn(Function):
    @staticmethod
    def forward(ctx, img, w, b, cls, pos, store):
        code = store.dtype
        Bn, _, H, W = img.shape
        E = w.shape[0]
        ntok = (H // 16) * (W // 16) + 1
        if pos.shape[1] != ntok:
            raise S4FError(f'pos_embed has {pos.shape[1]} tokens, input needs {ntok} (resize is an inference-only path)')
        cols = torch.zeros(Bn * ntok, 768, device=img.device, dtype=_T(code))
        K.im2col_patch16(img, cols, code, pad_cls=True)
        tokens = torch.empty(Bn, ntok, E, device=img.device, dtype=_R(code))
        posf = store.phys(pos)
        _gemm_resid(cols, store.shadow(w), Bn * ntok, E, 768, code, store.phys(b), None, tokens, pos_period=ntok, pos=posf)
        K.cls_pos(store.phys(cls), posf, tokens)
        ctx.store, ctx.cols, ctx.dims = store, cols, (Bn, ntok, E)
        ctx.prm = (w, b, cls, pos)
        return tokens

    @staticmethod
    def backward(ctx, dtok):
        store, cols = ctx.store, ctx.cols
        code = store.dtype
        Bn, ntok, E = ctx.dims
        w, b, cls, pos = ctx.prm
        dtok = dtok.contiguous()
        dt_t = dtok if dtok.dtype == _T(code) else _as_T(dtok, code)
        _wgrad(dt_t, cols, E, 768, Bn * ntok, E, 768, store.grad_phys(w), code)
        K.colsum(dtok, E, Bn * ntok, E, store.grad_phys(b), BF16 if dtok.dtype == torch.bfloat16 else F32, skip_period=ntok)
        K.tokens_bwd(dtok, store.grad_phys(pos), store.grad_phys(cls))
        ctx.cols = None
        store.node_done()
        return None, None, None, None, None, None



# ============================================================================================== fused layer launches (round 3)
# One C-ABI call per encoder-layer forward / backward (csrc/layer.hip) instead of one per kernel.  The per-kernel path below
# stays: it is what runs under the profiler (bench.py's per-GEMM roofline accounting needs one event pair per GEMM), with
# S4F_FUSED_LAUNCH=0, and for GEMM signatures the shipped tuning table does not know yet (they are tuned there on first use).
FUSED_LAUNCH = os.environ.get('S4F_FUSED_LAUNCH', '1') != '0'
# Round 4: attention backward as ONE sweep over the scores (s4f_attention_bwd_fused, bf16 mode; `=0`: the two-kernel form).  Its
# workspace (the fp32 dQ slabs: 204 MB at 16 images x 1025 tokens) is ONE buffer per device shared by all layers: the backward of
# the layers is serial on the chain's stream, and the buffer holds nothing between two calls.
ATTN_BWD_FUSED = os.environ.get('S4F_ATTN_BWD_FUSED', '1') != '0'
# Round 5: gelu'(z), the tensor the fc1 epilogue leaves for the backward, as 8-bit fixed point in bf16 mode (s4f_gemm_desc.gelu_q8:
# step 1/192 = what bf16 resolves near 1): 50 MB less written by fc1 and read by the fc2 input gradient per layer.  Round 6: OPT-IN
# (`S4F_GELU_Q8=1`).  The fixed step is an ABSOLUTE error of up to 1/384 whatever |gelu'| is - where |gelu'| is small (z < -2) that
# is 10 - 100 % relative and |gelu'| < 1/384 flushes to 0, where bf16 keeps 2^-9 relative - and its gain in the step (0.05 - 0.09 ms,
# profiles/r05_ab_gelu_q8.txt) is inside the run-to-run spread: a departure from the reference's numerics that buys nothing.
GELU_Q8 = os.environ.get('S4F_GELU_Q8', '0') != '0'
_ATTN_WS = {}


def _attn_bwd_ws(Bn, N, H, device):
    need = K.attention_bwd_ws_bytes(Bn, N, H)
    # one workspace per (device, STREAM): the buffer holds nothing between two calls, but two backward passes enqueued on different
    # streams (a second model, a backward under a head stream) would race on the dQ slabs of a shared one
    key = (device.type, device.index, torch.cuda.current_stream(device).cuda_stream)
    ws = _ATTN_WS.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.empty(need, device=device, dtype=torch.uint8)
        _ATTN_WS[key] = ws
    ws.record_stream(torch.cuda.current_stream(device))
    return ws

_LAYER_PLANS = {}

def _layer_plan(store, prm, M, E, F_, H, code, R):
    """static part of a layer's launch descriptor: parameter / shadow / gradient pointers and the tuned tile variants of its
    GEMMs; None when a signature is not in the tuning table yet (the per-kernel path then tunes it)"""
    import ctypes
    from . import _lib as L_
    (g1, b1, wqkv, bqkv, wo, bo, g2, b2, w1, bf1, w2, bf2) = prm
    key = (id(store), id(g1), M, code, R, store.flat.data_ptr(), 0 if store.flat_t is None else store.flat_t.data_ptr(),
           0 if store.grad is None else store.grad.data_ptr())
    plan = _LAYER_PLANS.get(key)
    if plan is not None:
        return plan
    rt = R == torch.bfloat16
    hints = [0] * 8
    wg = (0, max(1, round(256 / (K._t256(F_, E) * 2 + K._t256(3 * E, E) + K._t256(E, E)))))
    if code == BF16 and K.AUTOTUNE:
        def sig(N_, K_, act, f32o, to, resid):
            k = (K.OP_ROW, K.OP_ROW, M, N_, K_, K_, K_, None, act, False, f32o, to, resid, 1)
            return k + ('resid_t',) if (resid and rt) else k
        sigs = [sig(3 * E, E, K.ACT_NONE, False, True, False), sig(E, E, K.ACT_NONE, not rt, rt, True),
                sig(F_, E, K.ACT_GELU, False, True, False), sig(E, F_, K.ACT_NONE, not rt, rt, True),
                sig(F_, E, K.ACT_GELU_BWD, False, True, False), sig(E, F_, K.ACT_NONE, False, True, False),
                sig(E, E, K.ACT_NONE, False, True, False), sig(E, 3 * E, K.ACT_NONE, False, True, False)]
        for i, sg in enumerate(sigs):
            ch = K._tuned_lookup(sg)
            if ch is None:
                return None
            hints[i] = int(ch[0])
        ch = K._tuned_lookup(('wgrad_grouped', (F_, E, M), (E, F_, M), (3 * E, E, M), (E, E, M)))
        if ch is None:
            return None
        wg = (int(ch[0]), int(ch[1]))
    elif code == BF16:
        wg = (4, wg[1])
    if os.environ.get('S4F_WG_SPLITK'):      # experiment: k-ranges of the layer's grouped weight gradient (108 tiles x k-ranges blocks)
        wg = (wg[0], int(os.environ['S4F_WG_SPLITK']))
    if os.environ.get('S4F_WG_HINT'):        # experiment (round 5): tile variant of the layer's grouped weight gradient (2 = 256 x 128, 8 waves)
        wg = (int(os.environ['S4F_WG_HINT']), wg[1])
    d = L_.LayerDesc()
    d.E, d.F, d.H, d.dtype, d.xdtype = E, F_, H, code, (BF16 if rt else F32)
    for i in range(8):
        d.hint[i] = hints[i]
    d.wg_hint, d.wg_splitk, d.fold_colsum = wg[0], wg[1], 1 if K.FOLD_COLSUM else 0
    ph, gr, sh = store.phys, store.grad_phys, store.shadow
    for name, t in (('ln1_g', g1), ('ln1_b', b1), ('ln2_g', g2), ('ln2_b', b2), ('bqkv', bqkv), ('bo', bo), ('b1', bf1), ('b2', bf2)):
        setattr(d, name, ph(t).data_ptr())
    for name, t in (('wqkv', wqkv), ('wo', wo), ('w1', w1), ('w2', w2)):
        setattr(d, name, sh(t).data_ptr())
    if store.grad is not None:
        for name, t in (('d_ln1_g', g1), ('d_ln1_b', b1), ('d_ln2_g', g2), ('d_ln2_b', b2), ('d_wqkv', wqkv), ('d_bqkv', bqkv), ('d_wo', wo),
                        ('d_bo', bo), ('d_w1', w1), ('d_b1', bf1), ('d_w2', w2), ('d_b2', bf2)):
            setattr(d, name, gr(t).data_ptr())
    plan = dict(desc=d, T_set=False, event=None)
    _LAYER_PLANS[key] = plan
    return plan


def _plan_backward_ready(plan, store, prm, code, dev):
    """transposed weight shadows (bf16) registered / fresh, the fork event created"""
    (_, _, wqkv, _, wo, _, _, _, w1, _, w2, _) = prm
    d = plan['desc']
    if code == BF16:
        if not plan['T_set'] or not store._T_fresh or store._T_event is not None:
            for name, t in (('wqkv_T', wqkv), ('wo_T', wo), ('w1_T', w1), ('w2_T', w2)):
                setattr(d, name, store.shadow_T(t).data_ptr())          # (registers on first use, re-syncs / waits when stale)
            plan['T_set'] = True
    if plan['event'] is None:
        ev = torch.cuda.Event()
        ev.record()                                                      # instantiates the underlying hipEvent_t
        plan['event'] = ev
    return plan['event']


# ============================================================================================== options of the encoder layer
class LayerOpt:
    """What an encoder layer does beyond the reference's: norm - RMS norm of queries and keys per head (two gain parameters behind the
    layer's twelve); cos, sin - rotation of queries and keys by the position of their token ([tokens, 32] tables); q8 - the activations
    that only the backward pass reads are kept in 8 bits (kernels.act_pack) instead of their own type; grad - a backward pass may follow (the
    caller's grad mode: needs_input_grad tells only which inputs ask for gradients)."""
    __slots__ = ('norm', 'cos', 'sin', 'q8', 'grad')

    def __init__(self, norm=False, cos=None, sin=None, q8=False, grad=True):
        self.norm, self.cos, self.sin, self.q8, self.grad = norm, cos, sin, q8, grad

    @property
    def qk(self):
        return self.norm or self.cos is not None


class Packed:
    """an activation put away in 8 bits; restore() brings it back in its own type and shape"""
    __slots__ = ('codes', 'scales', 'shape', 'dtype')

    def __init__(self, t):
        self.shape, self.dtype = t.shape, t.dtype
        m = t.view(-1, t.shape[-1])
        self.codes = torch.empty(m.shape, device=t.device, dtype=torch.int8)
        self.scales = torch.empty(m.shape[0], m.shape[1] // 32, device=t.device, dtype=torch.uint8)
        K.act_pack(m, self.codes, self.scales, K._xcode(t))

    def restore(self):
        out = torch.empty(self.shape, device=self.codes.device, dtype=self.dtype)
        K.act_unpack(self.codes, self.scales, out.view(-1, self.shape[-1]), K._xcode(out))
        return out


def _restored(t):
    return t.restore() if isinstance(t, Packed) else t


def _project_qk(xn, w, b, qkv, M, E, H, code, eps, opt, gq, gk, store, keep):
    """qkv [M, 3 E] = the projection of xn with queries and keys normed / turned; returns what their backward reads: None, the pre-norm
    queries and keys, or (8-bit checkpoints) their codes and scales.  With a checkpoint, or when nothing is kept, the projection is one
    GEMM and the norm works in place; else queries and keys go to a tensor of their own, values straight to their place in qkv (no
    copy of the pre-norm tensor is made either way)."""
    par = dict(gq=store.phys(gq) if opt.norm else None, gk=store.phys(gk) if opt.norm else None, cos=opt.cos, sin=opt.sin, eps=eps)
    qk = qkv[:, :2 * E]
    wt = store.shadow(w)
    if keep and opt.norm and not opt.q8:
        pre = torch.empty(M, 2 * E, device=qkv.device, dtype=qkv.dtype)
        K.gemm(xn, wt[:2 * E * E], M, 2 * E, E, E, E, code, bias=b[:2 * E], out_t=pre, ldo_t=2 * E)
        K.gemm(xn, wt[2 * E * E:], M, E, E, E, E, code, bias=b[2 * E:], out_t=qkv.view(-1)[2 * E:], ldo_t=3 * E)
        K.qk_norm_rope_fwd(pre, qk, H, H, code, **par)
        return pre
    K.gemm(xn, wt, M, 3 * E, E, E, E, code, bias=b, out_t=qkv, ldo_t=3 * E)
    packed = None
    if keep and opt.norm:
        packed = (torch.empty(M, 2 * E, device=qkv.device, dtype=torch.int8), torch.empty(M, E // 16, device=qkv.device, dtype=torch.uint8))
    K.qk_norm_rope_fwd(qk, qk, H, H, code, packed=packed, **par)
    return packed


def _project_qk_bwd(dqkv, pre, M, E, H, code, eps, opt, gq, gk, store):
    """gradient of queries and keys in dqkv [M, 3 E] -> of the projection's outputs, in place; the gains' gradients into the arena"""
    dqk = dqkv[:, :2 * E]
    kw = {}
    if opt.norm:
        kw = dict(gq=store.phys(gq), gk=store.phys(gk), dgq=store.grad_phys(gq), dgk=store.grad_phys(gk),
                  ws=torch.empty(K.qk_norm_rope_ws_bytes(M, H, H), device=dqkv.device, dtype=torch.uint8))
        kw['packed' if isinstance(pre, tuple) else 'x'] = pre
    K.qk_norm_rope_bwd(dqk, dqk, H, H, code, cos=opt.cos, sin=opt.sin, eps=eps, **kw)


# ============================================================================================== encoder layer
class LayerFn(Function):
    """x [B,N,E] fp32 -> x + MHA(LN1(x)) -> (+ FFN(LN2(.)))   (vit.py:113-127)"""

    @staticmethod
    def forward(ctx, x, bias_u, row_flag, bias_w, num_heads, eps, store, opt, *prm):
        (g1, b1, wqkv, bqkv, wo, bo, g2, b2, w1, bf1, w2, bf2) = prm[:12]
        gq, gk = prm[12:] if opt is not None and opt.norm else (None, None)
        code = store.dtype
        T = _T(code)
        Bn, N, E = x.shape
        M = Bn * N
        F_ = w1.shape[0]
        dev = x.device
        x = x.contiguous()
        R = x.dtype
        need_grad = any(ctx.needs_input_grad) and (opt is None or opt.grad)
        if opt is not None and not (opt.qk or need_grad):
            opt = None                                       # checkpoints alone, and nothing to keep: the plain layer
        xn = torch.empty(M, E, device=dev, dtype=T)
        mean1 = torch.empty(M, device=dev); rstd1 = torch.empty(M, device=dev)
        qkv = torch.empty(M, 3 * E, device=dev, dtype=T)
        ctxv = torch.empty(M, E, device=dev, dtype=T)
        lse = torch.empty(Bn, num_heads, N, device=dev)
        x1 = torch.empty(Bn, N, E, device=dev, dtype=R)
        xn2 = torch.empty(M, E, device=dev, dtype=T)
        mean2 = torch.empty(M, device=dev); rstd2 = torch.empty(M, device=dev)
        # gelu'(z) is written only when a backward pass will read it (never on the teacher / inference path)
        q8 = opt is not None and opt.q8 and need_grad
        z = torch.empty(M, F_, device=dev, dtype=torch.uint8 if ((GELU_Q8 or q8) and code == BF16) else T) if need_grad else None
        a = torch.empty(M, F_, device=dev, dtype=T)
        x2 = torch.empty(Bn, N, E, device=dev, dtype=R)
        plan = _layer_plan(store, prm, M, E, F_, num_heads, code, R) if (FUSED_LAUNCH and L._prof is None and opt is None) else None
        pre = None
        if plan is not None:
            d = plan['desc']
            d.B, d.N, d.eps, d.bias_w = Bn, N, eps, float(bias_w)
            d.bias_u, d.row_flag = _lp(bias_u), _lp(row_flag)
            d.x, d.xn, d.mean1, d.rstd1, d.qkv, d.ctx, d.lse = x.data_ptr(), xn.data_ptr(), mean1.data_ptr(), rstd1.data_ptr(), qkv.data_ptr(), ctxv.data_ptr(), lse.data_ptr()
            d.x1, d.xn2, d.mean2, d.rstd2, d.gelu_d, d.a, d.x2 = x1.data_ptr(), xn2.data_ptr(), mean2.data_ptr(), rstd2.data_ptr(), _lp(z), a.data_ptr(), x2.data_ptr()
            d.gelu_q8 = 1 if (z is not None and z.dtype == torch.uint8) else 0
            L.call('s4f_encoder_layer_fwd', d, L.stream())
        else:
            K.layernorm_fwd(x, store.phys(g1), store.phys(b1), xn, mean1, rstd1, M, E, code, eps)
            if opt is not None and opt.qk:
                pre = _project_qk(xn, wqkv, store.phys(bqkv), qkv, M, E, num_heads, code, eps, opt, gq, gk, store, need_grad)
            else:
                K.gemm(xn, store.shadow(wqkv), M, 3 * E, E, E, E, code, bias=store.phys(bqkv), out_t=qkv, ldo_t=3 * E)
            K.attention_fwd(qkv, ctxv, lse, Bn, N, num_heads, code, bias_u=bias_u, row_flag=row_flag, bias_w=bias_w)
            _gemm_resid(ctxv, store.shadow(wo), M, E, E, code, store.phys(bo), x, x1)
            K.layernorm_fwd(x1, store.phys(g2), store.phys(b2), xn2, mean2, rstd2, M, E, code, eps)
            K.gemm(xn2, store.shadow(w1), M, F_, E, E, E, code, bias=store.phys(bf1), out_t=a, ldo_t=F_, out_pre=z, ldo_pre=F_ if need_grad else 0,
                   act=K.ACT_GELU)
            _gemm_resid(a, store.shadow(w2), M, E, F_, code, store.phys(bf2), x1, x2)
        if need_grad:
            ctx.store, ctx.prm = store, prm
            ctx.range = store.range_of(prm)
            store.range_acquire(ctx.range)
            ctx.cfg = (Bn, N, E, F_, num_heads, bias_w, eps, opt)
            if q8:
                # queries, keys and values stay in T: the attention backward recomputes the scores, and probabilities of perturbed
                # scores no longer sum to one against the saved log-sum-exp.  Statistics stay fp32
                x, xn, ctxv, x1, xn2, a = (Packed(t) for t in (x, xn, ctxv, x1, xn2, a))
                z = z if code == BF16 else Packed(z)
            ctx.sv = dict(x=x, xn=xn, mean1=mean1, rstd1=rstd1, qkv=qkv, ctxv=ctxv, lse=lse, x1=x1, xn2=xn2, mean2=mean2,
                          rstd2=rstd2, z=z, a=a, bias_u=bias_u, row_flag=row_flag, pre=pre)
        return x2

    @staticmethod
    def backward(ctx, g2):
        store = ctx.store
        code = store.dtype
        T = _T(code)
        (gm1, b1, wqkv, bqkv, wo, bo, gm2, b2, w1, bf1, w2, bf2) = ctx.prm[:12]
        Bn, N, E, F_, H, bias_w, eps, opt = ctx.cfg
        gq, gk = ctx.prm[12:] if opt is not None and opt.norm else (None, None)
        q8 = opt is not None and opt.q8
        sv = ctx.sv
        if sv is None:
            raise S4FError('backward of an encoder layer a second time: its saved activations are gone')
        M = Bn * N
        dev = g2.device
        g2 = g2.contiguous()
        R = g2.dtype                              # residual-stream type: the gradient stream has it too
        g2t = g2 if R == T else _as_T(g2, code)
        g2cs = _handed_colsum(g2)
        a_act, xn2, ctxv, xn = sv['a'], sv['xn2'], sv['ctxv'], sv['xn']
        dz = torch.empty(M, F_, device=dev, dtype=T)
        dxn2 = torch.empty(M, E, device=dev, dtype=T)
        g1 = torch.empty(Bn, N, E, device=dev, dtype=R)
        g1t = torch.empty(Bn, N, E, device=dev, dtype=T) if (code == BF16 and R != T) else g1
        dctx = torch.empty(M, E, device=dev, dtype=T)
        dqkv = torch.empty(M, 3 * E, device=dev, dtype=T)
        delta = torch.empty(Bn, H, N, device=dev)
        attn_ws = _attn_bwd_ws(Bn, N, H, dev) if (code == BF16 and ATTN_BWD_FUSED) else None
        dxn = torch.empty(M, E, device=dev, dtype=T)
        g0 = torch.empty(Bn, N, E, device=dev, dtype=R)
        g0t = torch.empty(Bn, N, E, device=dev, dtype=T) if (code == BF16 and R != T) else None
        g0cs = zeros_small(E, dev)
        plan = _layer_plan(store, ctx.prm, M, E, F_, H, code, R) if (FUSED_LAUNCH and L._prof is None and opt is None) else None
        if plan is not None:
            ev = _plan_backward_ready(plan, store, ctx.prm, code, dev)
            d = plan['desc']
            d.B, d.N, d.bias_w = Bn, N, float(bias_w)
            d.bias_u, d.row_flag = _lp(sv['bias_u']), _lp(sv['row_flag'])
            d.x, d.xn, d.mean1, d.rstd1, d.qkv, d.ctx, d.lse = sv['x'].data_ptr(), xn.data_ptr(), sv['mean1'].data_ptr(), sv['rstd1'].data_ptr(), sv['qkv'].data_ptr(), ctxv.data_ptr(), sv['lse'].data_ptr()
            d.x1, d.xn2, d.mean2, d.rstd2, d.gelu_d, d.a = sv['x1'].data_ptr(), xn2.data_ptr(), sv['mean2'].data_ptr(), sv['rstd2'].data_ptr(), sv['z'].data_ptr(), a_act.data_ptr()
            d.gelu_q8 = 1 if sv['z'].dtype == torch.uint8 else 0
            d.g2, d.g2t, d.g2cs = g2.data_ptr(), g2t.data_ptr(), _lp(g2cs)
            d.dz, d.dxn2, d.g1, d.g1t, d.dctx, d.dqkv, d.delta, d.dxn = dz.data_ptr(), dxn2.data_ptr(), g1.data_ptr(), g1t.data_ptr(), dctx.data_ptr(), dqkv.data_ptr(), delta.data_ptr(), dxn.data_ptr()
            d.g0, d.g0t, d.g0cs = g0.data_ptr(), (g0t if g0t is not None else g0).data_ptr(), g0cs.data_ptr()
            d.attn_ws, d.attn_ws_bytes = (attn_ws.data_ptr(), attn_ws.numel()) if attn_ws is not None else (None, 0)
            use_side = USE_SIDE_STREAM and LAYER_WG_SIDE
            side = side_stream(dev) if use_side else None
            L.call('s4f_encoder_layer_bwd', d, L.stream(), side.cuda_stream if side is not None else None, ev.cuda_event if side is not None else None)
            if side is not None:
                for t in (dqkv, xn, dz, xn2, g1t, ctxv, g2t, a_act):
                    t.record_stream(side)           # allocated on the chain's stream, read by the weight-gradient stream
            sv['z'] = sv['a'] = None
        else:
            # ---- FFN
            # The four weight gradients of the layer go out as ONE grouped launch on the side stream once the last operand
            # (dqkv) exists: alone each has 9..36 output tiles and needs a deep split-K; together they fill the chip.
            if g2cs is None:
                with on_side(dev, g2t):
                    K.colsum(g2t, E, M, E, store.grad_phys(bf2), code)
            else:
                store.grad_phys(bf2).add_(g2cs)
            # (the fc1 bias gradient = column sums of dz comes out of the GEMM's staged output tile where the variant allows)
            folded = _dgrad(g2t, w2, M, F_, E, store, code, out_t=dz, ldo_t=F_, aux=_restored(sv['z']), ld_aux=F_, act=K.ACT_GELU_BWD,
                            colsum=store.grad_phys(bf1))
            sv['z'] = sv['a'] = None
            if not folded:
                with on_side(dev, dz):
                    K.colsum(dz, F_, M, F_, store.grad_phys(bf1), code)
            _dgrad(dz, w1, M, E, F_, store, code, out_t=dxn2, ldo_t=E)
            # the column sums of g1 (= the proj bias gradient) come out of the same pass
            K.layernorm_bwd(dxn2, _restored(sv['x1']), sv['mean2'], sv['rstd2'], store.phys(gm2), g2, g1, g1t if g1t is not g1 else None, store.grad_phys(gm2),
                            store.grad_phys(b2), M, E, code, dcolsum=store.grad_phys(bo))
            # ---- attention
            _dgrad(g1t, wo, M, E, E, store, code, out_t=dctx, ldo_t=E)
            ctx_t = _restored(ctxv)
            if attn_ws is not None:
                K.attention_bwd_fused(sv['qkv'], ctx_t, dctx, sv['lse'], delta, dqkv, Bn, N, H, attn_ws, bias_u=sv['bias_u'],
                                      row_flag=sv['row_flag'], bias_w=bias_w)
            else:
                K.attention_bwd(sv['qkv'], ctx_t, dctx, sv['lse'], delta, dqkv, Bn, N, H, code, bias_u=sv['bias_u'],
                                row_flag=sv['row_flag'], bias_w=bias_w)
            del ctx_t
            if opt is not None and opt.qk:
                _project_qk_bwd(dqkv, sv['pre'], M, E, H, code, eps, opt, gq, gk, store)
            if q8:
                kept = ((dz, xn2, w1), (g2t, a_act, w2), (dqkv, xn, wqkv), (g1t, ctxv, wo))
                with on_side(dev, *[t for dy, pk, _ in kept for t in (dy, pk.codes, pk.scales)], enable=LAYER_WG_SIDE):
                    probs = [(dy.view(M, -1), pk.codes, pk.scales, store.grad_phys(w).view(w.shape)) for dy, pk, w in kept]
                    ws = torch.empty(K.wgrad_packed_ws_bytes([(*w.shape, M) for _, _, w in kept], code), device=dev, dtype=torch.uint8)
                    K.wgrad_packed(probs, code, ws)
                    K.colsum(dqkv, 3 * E, M, 3 * E, store.grad_phys(bqkv), code)
                    del ws, probs
            else:
                with on_side(dev, dqkv, xn, dz, xn2, g1t, ctxv, g2t, a_act, enable=LAYER_WG_SIDE):
                    K.wgrad_grouped([(dz, xn2, F_, E, M, store.grad_phys(w1)),
                                     (g2t, a_act, E, F_, M, store.grad_phys(w2)),
                                     (dqkv, xn, 3 * E, E, M, store.grad_phys(wqkv)),
                                     (g1t, ctxv, E, E, M, store.grad_phys(wo))], code)
                    K.colsum(dqkv, 3 * E, M, 3 * E, store.grad_phys(bqkv), code)
            _dgrad(dqkv, wqkv, M, E, 3 * E, store, code, out_t=dxn, ldo_t=E)
            K.layernorm_bwd(dxn, _restored(sv['x']), sv['mean1'], sv['rstd1'], store.phys(gm1), g1, g0, g0t, store.grad_phys(gm1),
                            store.grad_phys(b1), M, E, code, dcolsum=g0cs)
        del dqkv, dz
        # reused by the previous layer if autograd hands this very tensor through unmodified (autograd may
        # accumulate other branches into it in place: the version counter catches that)
        if g0t is not None:
            g0._s4f_t = (g0t, g0._version, g0.data_ptr())
        g0._s4f_colsum = (g0cs, g0._version, g0.data_ptr())
        ctx.sv = None
        store.node_done()
        store.range_release(ctx.range)
        return (g0,) + (None,) * (7 + len(ctx.prm))


# Round 5: heads advancing in lockstep (MultiHeadLossFn: the four auxiliary heads) issue their same-shape small convs - the
# 32 x 32 stage: forward, input gradient, weight gradient - as ONE grouped grid each (s4f_gemm_grouped) instead of one launch per
# head.  `=0`: one launch per head as before.
GROUP_SMALL_CONVS = os.environ.get('S4F_GROUP_SMALL_CONVS', '1') != '0'


# ============================================================================================== token un-shuffle
class TokenGatherFn(Function):
    """out.rows = tokens.rows[fwd]  over the flattened [B * (T + 1), E] token tensor: the decode head's un-shuffle of a
    patch-shuffled image (decode_head.py:186-212; augment.token_unshuffle_maps).  Backward = the gather with the inverse map."""

    @staticmethod
    def forward(ctx, tokens, fwd, bwd):
        tokens = tokens.contiguous()
        Bn, ntok, E = tokens.shape
        out = torch.empty_like(tokens)
        K.gather_rows(tokens, out, fwd, Bn * ntok, E)
        ctx.bwd = bwd
        return out

    @staticmethod
    def backward(ctx, g):
        g = g.contiguous()
        Bn, ntok, E = g.shape
        out = torch.empty_like(g)
        K.gather_rows(g, out, ctx.bwd, Bn * ntok, E)
        return out, None, None


# ============================================================================================== SETR-PUP head
def _world():
    return dist.get_world_size() if (dist.is_available() and dist.is_initialized()) else 1


class _Exchange:
    """SyncBN statistics exchange of one or several heads advancing in lockstep.  Every head takes its 2 C floats from ONE
    buffer per round (alloc), fills them, and yields; when all heads of the round have yielded, the buffer crosses the
    ranks in ONE all-reduce.  With a single head this is the plain per-layer all-reduce."""

    def __init__(self, nheads, world):
        self.n, self.world = nheads, world
        self.buf, self.i = None, 0
        self.gemms = []                               # (args, kwargs, side tensors or None) asked for in this round

    def gemm(self, *args, side=None, **kw):
        """a GEMM that the heads of a lockstep group issue TOGETHER (round 5): registered here, launched - as ONE grouped grid when
        several heads ask in the same round - when the generator yields 'gemm'.  side: tensors read by a launch that belongs on
        the weight-gradient stream."""
        self.gemms.append((args, kw, side))

    def flush_gemms(self):
        reqs, self.gemms = self.gemms, []
        if not reqs:
            return
        side = reqs[0][2]
        if side is not None:
            tens = [t for _, _, sd in reqs for t in sd]
            with on_side(tens[0].device, *tens):
                K.gemm_group([(a, kw) for a, kw, _ in reqs])
        else:
            K.gemm_group([(a, kw) for a, kw, _ in reqs])

    def alloc(self, size, dev):
        if self.buf is None or self.i >= self.n:
            self.buf, self.i = zeros_small(self.n * size, dev), 0
        v = self.buf[self.i * size:(self.i + 1) * size]
        self.i += 1
        return v

    @staticmethod
    def issue(buf):
        """sum over the ranks, in place, ordered on the current stream"""
        dist.all_reduce(buf)

    def reduce(self):
        if self.buf is None:
            return
        if self.world > 1:
            self.issue(self.buf)
        self.buf = None


def _drive(gens, ex):
    """advance the generators in lockstep: one ex.reduce() per round of yields; returns their return values"""
    out = [None] * len(gens)
    live = list(range(len(gens)))
    while live:
        nxt, kinds = [], set()
        for i in live:
            try:
                kinds.add(next(gens[i]))
                nxt.append(i)
            except StopIteration as e:
                out[i] = e.value
        if nxt:
            if len(nxt) != len(live) or len(kinds) != 1:
                raise S4FError('lockstep heads must have the same structure (SyncBN layers, grouped launches)')
            if 'gemm' in kinds:
                ex.flush_gemms()                      # the round's GEMM requests as one grouped launch
            else:
                ex.reduce()
        live = nxt
    return out


def head_forward(tokens, hp, store, training, save):
    world = _world() if (hp['sync_bn'] and training) else 1
    return _run_one(_head_forward_gen, tokens, hp, store, training, save, world=world)


def _run_one(gen_fn, *args, world):
    ex = _Exchange(1, world)
    return _drive([gen_fn(*args, ex)], ex)[0]


def _head_forward_gen(tokens, hp, store, training, save, ex):
    """LN -> [conv3x3 -> (Sync)BN -> ReLU -> up]*n -> conv_seg (before the last upsample) -> low-res logits.
    tokens: fp32 [B, T+1, E] (cls first; dropped here).  hp: dict with the head's parameters/buffers/config.
    Returns (logits_lo fp32 [B*h*w, LOGIT_LD], (B, h, w), saved or None)."""
    code = store.dtype
    T = _T(code)
    Bn, ntok, E = tokens.shape
    dev = tokens.device
    gh, gw = hp['grid']
    if gh * gw + 1 != ntok:
        raise S4FError(f'head: token count {ntok} does not match the patch grid {gh}x{gw}')
    rows = Bn * gh * gw
    xn = torch.empty(rows, E, device=dev, dtype=T)
    mean0 = torch.empty(rows, device=dev); rstd0 = torch.empty(rows, device=dev)
    tv = tokens[:, 1:]
    K.layernorm_fwd(tv, store.phys(hp['norm_w']), store.phys(hp['norm_b']), xn, mean0, rstd0, rows, E, code, hp['ln_eps'],
                    rows_per_img=gh * gw, in_batch_stride=ntok * E)
    sv = dict(tokens=tokens, mean0=mean0, rstd0=rstd0, stages=[]) if save else None
    cur, h, w, cin = xn, gh, gw, E
    nconv = len(hp['convs'])
    logits = None
    world = _world() if (hp['sync_bn'] and training) else 1
    for k, cv in enumerate(hp['convs']):
        Cc = cv['w'].shape[0]
        Mp = Bn * h * w
        y = torch.empty(Mp, Cc, device=dev, dtype=T)
        sums, stats_done = None, False
        last_f32 = (TEACHER_LAST_FP32 and code == BF16 and k == nconv - 1 and not save and not training and FUSE_CLS_FWD
                    and Cc % 32 == 0 and Cc <= 512 and hp['num_classes'] <= 32)
        if last_f32:
            y = torch.empty(Mp, Cc, device=dev)
            K.gemm(cur, store.shadow(cv['w']), Mp, Cc, 9 * cin, cin, 9 * cin, code, a_mode=K.OP_ROW_CONV, out_f32=y, ldo_f32=Cc,
                   conv=(Bn, h, w, cin, 1))
        elif code == BF16 and _tiles256(Mp, Cc) < 96:
            # few output tiles (the 32x32 stage): split the 9*cin contraction over blocks, fp32 partial sums
            yf = torch.zeros(Mp, Cc, device=dev)
            if GROUP_SMALL_CONVS and ex.n > 1:
                # lockstep heads: the same-shape convs of all of them as ONE grid (s4f_gemm_grouped, 8-wave kernel, the k-ranges
                # sized for the group: n x tiles x splits ~ one block per CU)
                ex.gemm(cur, store.shadow(cv['w']), Mp, Cc, 9 * cin, cin, 9 * cin, code, a_mode=K.OP_ROW_CONV, out_f32=yf, ldo_f32=Cc,
                        atomic=True, splitk=max(1, min(16, 256 // (ex.n * _tiles256(Mp, Cc)))), conv=(Bn, h, w, cin, 1), tile_hint=10)
                yield 'gemm'
            else:
                K.gemm(cur, store.shadow(cv['w']), Mp, Cc, 9 * cin, cin, 9 * cin, code, a_mode=K.OP_ROW_CONV, out_f32=yf,
                       ldo_f32=Cc, atomic=True, splitk=max(2, min(16, 192 // _tiles256(Mp, Cc))), conv=(Bn, h, w, cin, 1))
            K.cast(yf, y, code)
        else:
            # training: the BatchNorm statistics (column sums and sums of squares of y as stored) come out of the conv GEMM's
            # staged output tile where the chosen kernel variant can do that (the two large stages), else from a pass over y
            sums = ex.alloc(2 * Cc, dev) if training else None
            stats_done = K.gemm(cur, store.shadow(cv['w']), Mp, Cc, 9 * cin, cin, 9 * cin, code, a_mode=K.OP_ROW_CONV, out_t=y,
                                ldo_t=Cc, conv=(Bn, h, w, cin, 1), colstats=sums)
        scale = torch.empty(Cc, device=dev); shift = torch.empty(Cc, device=dev)
        mean = torch.empty(Cc, device=dev); rstd = torch.empty(Cc, device=dev)
        count = float(Mp) * world
        if training:
            if sums is None:
                sums = ex.alloc(2 * Cc, dev)
            if not stats_done:
                K.bn_stats(y, Mp, Cc, sums, code)
            yield                                            # the statistics cross the ranks (lockstep heads: together)
            K.bn_finalize(sums, count, store.phys(cv['bn_w']), store.phys(cv['bn_b']), store.phys(cv['rm']),
                          store.phys(cv['rv']), hp['bn_momentum'], hp['bn_eps'], True, scale, shift, mean, rstd, Cc)
            cv['nbt'][0] += 1
        else:
            K.bn_finalize(None, 0, store.phys(cv['bn_w']), store.phys(cv['bn_b']), store.phys(cv['rm']),
                          store.phys(cv['rv']), hp['bn_momentum'], hp['bn_eps'], False, scale, shift, mean, rstd, Cc)
        s = hp['up_scale'] if k < nconv - 1 else 1
        if k == nconv - 1 and FUSE_CLS_FWD and Cc % 32 == 0 and Cc <= 512 and hp['num_classes'] <= 32 and LOGIT_LD >= 32:
            # last stage: BN affine + ReLU + conv_seg in ONE pass over y; the activation is written only if a backward
            # pass will need it (the conv_seg weight gradient), never on the teacher / inference path
            logits = torch.empty(Mp, LOGIT_LD, device=dev)
            # ... and not even then when the backward's statistics pass forms the conv_seg weight gradient from the activation
            # it rebuilds (FUSE_CLS_WGRAD)
            keep_u = save and not (FUSE_CLS_WGRAD and _fuse_cls_ok(s, Cc, hp['num_classes']))
            u = torch.empty(Mp, Cc, device=dev, dtype=T) if keep_u else None
            if last_f32:
                K.bn_relu_cls_fwd(y, scale, shift, store.phys(hp['seg_w']), store.phys(hp['seg_b']), logits, LOGIT_LD, None, Mp, Cc,
                                  hp['num_classes'], 0)
            else:
                K.bn_relu_cls_fwd(y, scale, shift, store.shadow(hp['seg_w']), store.phys(hp['seg_b']), logits, LOGIT_LD, u, Mp, Cc,
                                  hp['num_classes'], code)
        else:
            u = torch.empty(Bn * h * s * w * s, Cc, device=dev, dtype=T)
            K.bn_relu_up_fwd(y, scale, shift, u, Bn, h, w, Cc, s, code)
        if save:
            sv['stages'].append(dict(inp=cur, y=y, scale=scale, shift=shift, mean=mean, rstd=rstd, h=h, w=w, s=s, cin=cin,
                                     count=count, Cc=Cc))
        cur, h, w, cin = u, h * s, w * s, Cc
    ncls = hp['num_classes']
    Mp = Bn * h * w
    if logits is None:
        logits = torch.zeros(Mp, LOGIT_LD, device=dev)
        K.gemm(cur, store.shadow(hp['seg_w']), Mp, ncls, cin, cin, cin, code, bias=store.phys(hp['seg_b']), out_f32=logits,
               ldo_f32=LOGIT_LD)
    if save:
        sv['feat'] = cur
        sv['logits'] = logits
    return logits, (Bn, h, w), sv


def _fuse_cls_ok(s_last, Cc, ncls):
    return bool(FUSE_CLS_GRAD and SKIP_MASKED_COPY and s_last == 1 and Cc in (64, 128, 192, 256) and ncls <= 32 and LOGIT_LD >= 32)


def _fuse_cls_grad(sv, hp):
    """is the input gradient of conv_seg recomputed inside the last stage's two BN backward passes (cls_bn_bwd_stats / _apply)?
    Then nothing reads the fp32 gradient of the low-res logits, only its T copy - and (FUSE_CLS_WGRAD) the statistics pass also
    forms the conv_seg WEIGHT gradient from the activation it rebuilds, so that the forward does not store it (sv['feat'] None)."""
    last = sv['stages'][-1]
    return _fuse_cls_ok(last['s'], last['Cc'], hp['num_classes'])


def head_backward(dlo, dlo_t, sv, hp, store):
    """gradients of everything upstream of the low-res logits; returns d tokens (fp32 [B, T+1, E])."""
    return _run_one(_head_backward_gen, dlo, dlo_t, sv, hp, store, world=_world() if hp['sync_bn'] else 1)


def _head_backward_gen(dlo, dlo_t, sv, hp, store, ex):
    code = store.dtype
    T = _T(code)
    tokens = sv['tokens']
    Bn, ntok, E = tokens.shape
    dev = tokens.device
    ncls = hp['num_classes']
    feat = sv['feat']
    last = sv['stages'][-1]
    cin = last['Cc']
    Mp = Bn * last['h'] * last['s'] * last['w'] * last['s']
    # conv_seg: dW[ncls, cin] += dlo^T feat ; db += colsum(dlo) ; dfeat = dlo W
    wgrad_in_stats = feat is None
    if not wgrad_in_stats:
        K.gemm(dlo_t, feat, ncls, cin, Mp, LOGIT_LD, cin, code, a_mode=K.OP_K, b_mode=K.OP_K, out_f32=store.grad_phys(hp['seg_w']),
               ldo_f32=cin, atomic=True, splitk=_splitk(_tiles(ncls, cin), _nk(Mp, code), target=1024))
    # The input gradient of conv_seg, dfeat = dlo W, is not materialised when the stage below is the usual conv -> BN -> ReLU
    # without upsample: its two BN backward passes recompute it from the 32-column dlo rows on the matrix cores
    # (s4f_cls_bn_bwd_stats / _apply; FUSE_CLS_GRAD=0: the GEMM + the generic passes); the statistics pass also leaves the
    # conv_seg bias gradient (column sums of dlo)
    fuse_cls = _fuse_cls_grad(sv, hp)
    if wgrad_in_stats and not fuse_cls:
        raise S4FError('head backward: the forward did not keep the last activation but the fused conv_seg gradient is off')
    dcur = None
    if not fuse_cls:
        K.colsum(dlo, LOGIT_LD, Mp, ncls, store.grad_phys(hp['seg_b']), F32)
        dcur = torch.empty(Mp, cin, device=dev, dtype=T)
        K.gemm(dlo_t, store.shadow(hp['seg_w']), Mp, cin, ncls, LOGIT_LD, cin, code, b_mode=K.OP_K, out_t=dcur, ldo_t=cin)
    world = _world() if hp['sync_bn'] else 1
    for k in range(len(hp['convs']) - 1, -1, -1):
        cv, st = hp['convs'][k], sv['stages'][k]
        Cc, h, w, s, cin_k = st['Cc'], st['h'], st['w'], st['s'], st['cin']
        Mk = Bn * h * w
        bsums = ex.alloc(2 * Cc, dev)
        dy = torch.empty(Mk, Cc, device=dev, dtype=T)
        if dcur is None:
            K.cls_bn_bwd_stats(dlo_t, LOGIT_LD, store.shadow(hp['seg_w']), st['y'], st['scale'], st['shift'], st['mean'],
                               st['rstd'], bsums, Mk, Cc, ncls, code, seg_b_grad=store.grad_phys(hp['seg_b']),
                               seg_w_grad=store.grad_phys(hp['seg_w']) if wgrad_in_stats else None)
            K.bn_param_grads(bsums, store.grad_phys(cv['bn_w']), store.grad_phys(cv['bn_b']), Cc)
            yield                                            # the sums cross the ranks (lockstep heads: together)
            K.cls_bn_bwd_apply(dlo_t, LOGIT_LD, store.shadow(hp['seg_w']), st['y'], st['scale'], st['shift'], st['mean'],
                               st['rstd'], store.phys(cv['bn_w']), bsums, st['count'], dy, Mk, Cc, ncls, code)
            g = None
        elif s == 1 and SKIP_MASKED_COPY:
            # no upsample: the masked gradient g = dcur * relu' is not materialised; the statistics pass and the apply pass
            # both read (dcur, y) and re-mask on the fly
            K.bn_relu_up_bwd(dcur, st['y'], st['scale'], st['shift'], st['mean'], st['rstd'], None, bsums, Bn, h, w, Cc, 1, code)
            g, rs, rb = dcur, st['scale'], st['shift']
        else:
            g = torch.empty(Mk, Cc, device=dev, dtype=T)
            K.bn_relu_up_bwd(dcur, st['y'], st['scale'], st['shift'], st['mean'], st['rstd'], g, bsums, Bn, h, w, Cc, s, code)
            rs = rb = None
        if dcur is not None:
            K.bn_param_grads(bsums, store.grad_phys(cv['bn_w']), store.grad_phys(cv['bn_b']), Cc)
            yield                                            # the sums cross the ranks (lockstep heads: together)
            K.bn_bwd_apply(g, st['y'], st['mean'], st['rstd'], store.phys(cv['bn_w']), bsums, st['count'], dy, Mk, Cc, code,
                           relu_scale=rs, relu_shift=rb)
        del g
        st['y'] = None
        # conv weight gradient [Cc][3][3][cin] += dy^T (shifted inp)
        small = GROUP_SMALL_CONVS and ex.n > 1 and code == BF16 and _tiles256(Mk, cin_k) < 128 and cin_k % 256 == 0
        if small:
            ex.gemm(dy, st['inp'], Cc, 9 * cin_k, Mk, Cc, cin_k, code, a_mode=K.OP_K, b_mode=K.OP_K_CONV,
                    out_f32=store.grad_phys(cv['w']), ldo_f32=9 * cin_k, atomic=True,
                    splitk=max(1, min(_nk(Mk, code), 256 // (ex.n * _tiles256(Cc, 9 * cin_k)))), conv=(Bn, h, w, cin_k, 1), tile_hint=10,
                    side=(dy, st['inp']))
            yield 'gemm'
        else:
            with on_side(dev, dy, st['inp']):
                K.gemm(dy, st['inp'], Cc, 9 * cin_k, Mk, Cc, cin_k, code, a_mode=K.OP_K, b_mode=K.OP_K_CONV,
                       out_f32=store.grad_phys(cv['w']), ldo_f32=9 * cin_k, atomic=True,
                       splitk=_splitk(_tiles(Cc, 9 * cin_k), _nk(Mk, code), target=768), conv=(Bn, h, w, cin_k, 1))
        st['inp'] = None
        dcur = torch.empty(Mk, cin_k, device=dev, dtype=T)
        # input gradient = the same implicit GEMM with mirrored taps (csign -1).  bf16: against the [ci][tap][co] shadow
        # (row-major B, the forward kernel forms); fp32: the stored [co][tap][ci] weights read tap-split k-major.
        if code == BF16:
            wB, bm, ldb = store.shadow_T(cv['w']), K.OP_ROW, 9 * Cc
        else:
            wB, bm, ldb = store.shadow(cv['w']), K.OP_K_TAPSPLIT, 9 * cin_k
        if code == BF16 and _tiles256(Mk, cin_k) < 128:
            df = torch.zeros(Mk, cin_k, device=dev)
            if small:
                ex.gemm(dy, wB, Mk, cin_k, 9 * Cc, Cc, ldb, code, a_mode=K.OP_ROW_CONV, b_mode=bm, out_f32=df, ldo_f32=cin_k,
                        atomic=True, splitk=max(1, min(8, 256 // (ex.n * _tiles256(Mk, cin_k)))), conv=(Bn, h, w, Cc, -1), tile_hint=10)
                yield 'gemm'
            else:
                K.gemm(dy, wB, Mk, cin_k, 9 * Cc, Cc, ldb, code, a_mode=K.OP_ROW_CONV, b_mode=bm, out_f32=df, ldo_f32=cin_k,
                       atomic=True, splitk=max(2, min(8, 256 // _tiles256(Mk, cin_k))), conv=(Bn, h, w, Cc, -1))
            K.cast(df, dcur, code)
        else:
            K.gemm(dy, wB, Mk, cin_k, 9 * Cc, Cc, ldb, code, a_mode=K.OP_ROW_CONV, b_mode=bm, out_t=dcur, ldo_t=cin_k,
                   conv=(Bn, h, w, Cc, -1))
        del dy
    gh, gw = hp['grid']
    td = getattr(tokens, '_s4f_tapdst', None)        # (holder, group): this call's rows of the tap's shared gradient buffer
    acc = False
    if td is not None and td[0].buf is not None:
        dtok, acc = td[0].claim(td[1])
    else:
        td = None
        dtok = torch.empty(Bn, ntok, E, device=dev, dtype=tokens.dtype)
    if not acc:
        dtok[:, 0].zero_()                           # the head drops the cls row: only it needs zeros, the rest is written below
    K.layernorm_bwd(dcur, tokens[:, 1:], sv['mean0'], sv['rstd0'], store.phys(hp['norm_w']), None, dtok[:, 1:], None,
                    store.grad_phys(hp['norm_w']), store.grad_phys(hp['norm_b']), Bn * gh * gw, E, code,
                    rows_per_img=gh * gw, in_batch_stride=ntok * E, accumulate=acc)
    if td is not None:
        td[0].done(td[1])
    return None if acc else dtok                     # accumulated into another call's rows: nothing for autograd to add


class _TapGrad:
    """The gradient of ONE backbone tap (token tensor [B, T+1, E]) that several head calls consume by image group
    (labelled rows, pseudo-labelled rows, ...).  autograd's own plumbing for `tokens[a:b]` costs, per group and tap, a
    full-size zero fill, a copy into the slice and full-size additions (about 30 ATen launches and 0.3 ms at the head of
    the backbone's backward, profiles/r03_serial_launch_list.txt).  Here the heads' last backward kernel (the LayerNorm
    backward) writes its rows of ONE buffer directly; a second head on the same rows (decode head and fourth auxiliary
    head share the last tap) accumulates into them behind the first one's event and hands autograd no tensor at all."""

    def __init__(self, tokens, bounds):
        self.bounds = bounds
        self.buf = torch.empty_like(tokens)      # (on the forward's stream; the heads' streams only write into it)
        self.claims = {}                         # group index -> events of the writers so far

    def claim(self, gi):
        a, b = self.bounds[gi]
        evs = self.claims.get(gi)
        if evs is None:
            self.claims[gi] = []
            return self.buf[a:b], False
        torch.cuda.current_stream().wait_event(evs[-1])
        return self.buf[a:b], True

    def done(self, gi):
        ev = torch.cuda.Event()
        ev.record()
        self.claims[gi].append(ev)


class TapSplitFn(Function):
    """tokens [B, T+1, E] -> (tokens for the next encoder layer if `chain`,) + the views tokens[a:b] of the image groups;
    backward: see _TapGrad.  With the chain output the tap's gradient is added IN PLACE into the rows of the chain's gradient
    that some head covers (rows without a head get nothing: no zero fill, no full-size addition by autograd)."""

    @staticmethod
    def forward(ctx, tokens, holder, chain):
        ctx.holder, ctx.chain = holder, chain
        ctx.set_materialize_grads(False)
        parts = tuple(tokens[a:b] for a, b in holder.bounds)
        return ((tokens.view_as(tokens),) + parts) if chain else parts

    @staticmethod
    def backward(ctx, *grads):
        h = ctx.holder
        buf, cur = h.buf, torch.cuda.current_stream()
        dchain = None
        if ctx.chain:
            dchain, grads = grads[0], grads[1:]
        rows = set()
        ready = []                                   # groups whose rows of buf are complete
        for gi, (a, b) in enumerate(h.bounds):
            g, evs = grads[gi], h.claims.get(gi)
            if evs is None:                          # no head wrote these rows in place
                if g is None:
                    continue
                buf[a:b].copy_(g)
            else:
                for ev in evs:
                    cur.wait_event(ev)
                if g is not None and g.data_ptr() != buf[a:b].data_ptr():
                    # a consumer outside the protocol BESIDES heads that wrote in place: autograd has summed their view of buf with
                    # the other gradient out of place, so g already contains buf's rows - adding it would count the heads twice,
                    # copying it would be right only if every head had finished before autograd summed.  Not a case the step has.
                    raise S4FError('TapSplitFn: a tap part feeds both a head (in-place gradient) and another consumer; route the '
                                   'other consumer through its own part or set S4F_TAP_SPLIT=0')
            rows.update(range(a, b))
            ready.append((a, b))
        h.buf = None
        if dchain is not None:
            if dchain.dtype != buf.dtype:
                raise S4FError('tap gradient and chain gradient differ in type')
            if buf.dtype == torch.float32 and dchain.is_contiguous():
                # the layer behind this tap left the operand-typed copy and the column sums of its gradient ON the tensor
                # (LayerFn.backward: _s4f_t, _s4f_colsum, valid for the tensor's version): the copy is kept in step by the same
                # pass, the column sums are dropped (the layer in front then sums the columns itself, as it did when autograd's
                # addition handed it a fresh tensor).  Raw-pointer writes do not move the version counter.
                tt = getattr(dchain, '_s4f_t', None)
                g0t = tt[0] if tt is not None and tt[1] == dchain._version and tt[2] == dchain.data_ptr() else None
                for a, b in ready:                   # (groups do not overlap)
                    K.add_f32(dchain[a:b], buf[a:b], dchain[a:b], None if g0t is None else g0t[a:b], F32 if g0t is None else BF16)
                if ready:
                    dchain._s4f_colsum = None
                    if g0t is None:
                        dchain._s4f_t = None
            else:
                for a, b in ready:
                    dchain[a:b].add_(buf[a:b])       # (moves the version counter: what the layer left on the tensor lapses)
            return dchain, None, None
        for i in range(buf.shape[0]):
            if i not in rows:
                buf[i].zero_()                       # images no group covers
        return buf, None, None


HEAD_MARKS = None              # diagnostic (tools/exp/head_marks.py): list of (label, stream id, start event, end event, host t0, host t1)


def _mark_begin(label):
    if HEAD_MARKS is None:
        return None
    import time
    ev = torch.cuda.Event(enable_timing=True)
    ev.record()
    return (label, ev, time.perf_counter())


def _mark_end(m):
    if m is None:
        return
    import time
    ev = torch.cuda.Event(enable_timing=True)
    ev.record()
    HEAD_MARKS.append((m[0], torch.cuda.current_stream().cuda_stream, m[1], ev, m[2], time.perf_counter()))


class HeadLossFn(Function):
    """loss = loss_weight * mean_all_pixels CE(up_s(logits_lo), labels; ignore 255)   (Q5)
    With ncr_lo (the teacher's low-resolution logits of the same images): returns (loss, loss_ncr), loss_ncr = the negative
    class ranking term of encoder_decoder.py:936-954 (mode 'unsup_only') on the SAME student logits; the backward adds both
    gradients on the low-resolution logits before the head's backward runs once."""

    @staticmethod
    def forward(ctx, tokens, labels_u8, loss_weight, hp, store, ncr_lo, *prm):
        need_grad = any(ctx.needs_input_grad)
        mk = _mark_begin(('fwd', len(hp['convs']), int(tokens.shape[0])))
        logits, (Bn, h, w), sv = head_forward(tokens, hp, store, training=hp['training'], save=need_grad)
        s = hp['up_scale']
        H, W = h * s, w * s
        if tuple(labels_u8.shape) != (Bn, H, W):
            raise S4FError(f'labels {tuple(labels_u8.shape)} do not match the logits size {(Bn, H, W)} '
                           '(the identity resize of decode_head.py:322-326 is the only one on the hot path)')
        loss_sum = zeros_small(1, tokens.device)
        # logsumexp per pixel is kept for the backward (4 B / pixel) so that it does not re-normalise the softmax
        lse = torch.empty(Bn, H, W, device=tokens.device) if need_grad and s in (2, 4) else None
        K.upce_fwd(logits, labels_u8, loss_sum, Bn, h, w, hp['num_classes'], LOGIT_LD, s, hp['ignore_index'], lse_out=lse)
        k = float(loss_weight) / float(Bn * H * W)
        if need_grad:
            ctx.sv, ctx.hp, ctx.store = sv, hp, store
            ctx.meta = (labels_u8, k, Bn, h, w, s)
            ctx.lse = lse
            ctx.consumer = GRAD_CONSUMER
            # a head may be called several times per step (decode head: labelled + pseudo-labelled batch); its arena range
            # is final - and handed to the gradient reducer - when the last of those calls has run its backward
            ctx.range = store.range_of(prm)
            store.range_acquire(ctx.range)
            ctx.ncr_lo = ncr_lo
        loss = (loss_sum * k).reshape(())
        _mark_end(mk)
        if ncr_lo is None:
            return loss
        ncr_sum = zeros_small(1, tokens.device)
        K.ncr_fwd(logits, ncr_lo, labels_u8, ncr_sum, Bn, h, w, hp['num_classes'], LOGIT_LD, s)
        return loss, (ncr_sum * (1.0 / float(Bn * H * W))).reshape(())

    @staticmethod
    def backward(ctx, dloss, dncr=None):
        sv, hp, store = ctx.sv, ctx.hp, ctx.store
        labels, k, Bn, h, w, s = ctx.meta
        code = store.dtype
        logits = sv['logits']
        mk = _mark_begin(('bwd', len(hp['convs']), int(Bn)))
        dlo_t = torch.empty(logits.shape, device=logits.device, dtype=torch.bfloat16) if code == BF16 else None
        # bf16 mode with the fused conv_seg gradient: nothing reads the fp32 gradient of the logits, only its T copy
        t_only = dlo_t is not None and ctx.lse is not None and _fuse_cls_grad(sv, hp) and not (ctx.ncr_lo is not None and dncr is not None)
        dlo = None if t_only else torch.empty_like(logits)
        gdev = dloss.detach().reshape(1).to(torch.float32).contiguous()
        K.upce_bwd(logits, labels, k, dlo, dlo_t, Bn, h, w, hp['num_classes'], LOGIT_LD, s, code, hp['ignore_index'],
                   gscale_dev=gdev, lse=ctx.lse)
        ctx.lse = None
        if ctx.ncr_lo is not None and dncr is not None:
            ndev = dncr.detach().reshape(1).to(torch.float32).contiguous()
            K.ncr_bwd(logits, ctx.ncr_lo, labels, 1.0 / float(Bn * h * s * w * s), dlo, dlo_t, Bn, h, w, hp['num_classes'], LOGIT_LD,
                      s, code, gscale_dev=ndev)
        ctx.ncr_lo = None
        dtok = head_backward(dlo, dlo_t if dlo_t is not None else dlo, sv, hp, store)
        _mark_end(mk)
        if ctx.consumer is not None and dtok is not None:
            dtok.record_stream(ctx.consumer)          # allocated on the head's stream, read by the backbone's
        ctx.sv = None
        store.node_done()
        store.range_release(ctx.range)
        return (dtok, None, None, None, None, None) + (None,) * (len(ctx.needs_input_grad) - 6)


class MultiHeadLossFn(Function):
    """The fused losses of several structurally identical head CALLS (the four auxiliary heads; the decode head's labelled
    and pseudo-labelled calls) advancing in LOCKSTEP: layer k of every call, then ONE SyncBN all-reduce for all of them,
    instead of one per call and layer (32 -> 12 exchanges per step; each exchange is a round trip between the head's
    stream and RCCL's).  Per call the arithmetic, the kernels and their order are those of HeadLossFn; calls of the SAME
    head update its BN running statistics layer by layer in call order, as consecutive calls do."""

    @staticmethod
    def forward(ctx, store, metas, *tensors):
        n = len(metas)                                   # metas[i] = (loss_weight, hp, number of parameters, labels u8)
        tokens = tensors[:n]
        need_grad = any(ctx.needs_input_grad)
        world = _world() if (metas[0][1]['sync_bn'] and metas[0][1]['training']) else 1
        ex = _Exchange(n, world)
        labels_u8 = None
        outs = _drive([_head_forward_gen(tokens[i], metas[i][1], store, metas[i][1]['training'], need_grad, ex)
                       for i in range(n)], ex)
        losses, saved = [], []
        off = n
        for i in range(n):
            lw, hp, nprm, labels_u8 = metas[i]
            logits, (Bn, h, w), sv = outs[i]
            s = hp['up_scale']
            H, W = h * s, w * s
            if tuple(labels_u8.shape) != (Bn, H, W):
                raise S4FError(f'labels {tuple(labels_u8.shape)} do not match the logits size {(Bn, H, W)}')
            loss_sum = zeros_small(1, tokens[i].device)
            lse = torch.empty(Bn, H, W, device=tokens[i].device) if need_grad and s in (2, 4) else None
            K.upce_fwd(logits, labels_u8, loss_sum, Bn, h, w, hp['num_classes'], LOGIT_LD, s, hp['ignore_index'], lse_out=lse)
            k = float(lw) / float(Bn * H * W)
            losses.append((loss_sum * k).reshape(()))
            if need_grad:
                rng = store.range_of(tensors[off:off + nprm])
                store.range_acquire(rng)
                saved.append(dict(sv=sv, hp=hp, meta=(k, Bn, h, w, s), lse=lse, labels=labels_u8, range=rng))
            off += nprm
        if need_grad:
            ctx.saved, ctx.store, ctx.n = saved, store, n
            ctx.consumer = GRAD_CONSUMER
        return tuple(losses)

    @staticmethod
    def backward(ctx, *dlosses):
        store, n = ctx.store, ctx.n
        code = store.dtype
        gens = []
        for i in range(n):
            sd = ctx.saved[i]
            sv, hp = sd['sv'], sd['hp']
            k, Bn, h, w, s = sd['meta']
            logits = sv['logits']
            dlo = torch.empty_like(logits)
            dlo_t = torch.empty(logits.shape, device=logits.device, dtype=torch.bfloat16) if code == BF16 else None
            gdev = dlosses[i].detach().reshape(1).to(torch.float32).contiguous()
            K.upce_bwd(logits, sd['labels'], k, dlo, dlo_t, Bn, h, w, hp['num_classes'], LOGIT_LD, s, code, hp['ignore_index'],
                       gscale_dev=gdev, lse=sd['lse'])
            sd['lse'] = None
            gens.append((dlo, dlo_t if dlo_t is not None else dlo, sv, hp))
        world = _world() if ctx.saved[0]['hp']['sync_bn'] else 1
        ex = _Exchange(n, world)
        dtoks = _drive([_head_backward_gen(a, b, sv, hp, store, ex) for a, b, sv, hp in gens], ex)
        for i in range(n):
            if ctx.consumer is not None and dtoks[i] is not None:
                dtoks[i].record_stream(ctx.consumer)
            store.node_done()
            store.range_release(ctx.saved[i]['range'])
        ctx.saved = None
        return (None, None) + tuple(dtoks) + (None,) * (len(ctx.needs_input_grad) - 2 - n)
