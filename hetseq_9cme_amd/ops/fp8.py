"""8-bit training: linear layers on e4m3 operands, activations kept in 8 bits for the backward.

A block is 128 consecutive entries sharing one power-of-two scale 2^e (csrc/include/hx_quant.h):

* e4m3 (operands of products): e the smallest integer with max |x| <= 448 2^e, code = e4m3(x 2^-e);
* int8 (kept activations):     e the smallest integer with max |x| <= 127 2^e, code = rint(x 2^-e),

both rounded to nearest even; e = 0 for a block of zeros, e >= -126.  Entries that are not finite do
not take part in the maximum and come back as NaN, so an overflow still reaches the loss and the
gradient norm.  A power of two costs at most one bit of a block's range and rounds nothing itself,
so codes are the same bits whatever computes them.

``linear_fp8`` blocks every operand along the dimension its product sums over:

    y  = Q(x)  Q(W)^T + b      blocks along the input features
    dx = Q(dy) Q(W^T)^T        blocks along the output features
    dW = Q(dy^T) Q(x^T)^T      blocks along the tokens
    db = sum of dy's rows      (not rounded)

What it keeps for the backward is Q(x^T): one byte per element (and 1 / 128) instead of two or four.
Results in bf16 come from the matrix cores' scaled e4m3 instructions, results in fp32 (dW, and y / dx
of fp32 activations) from exact bf16 copies of the codes (csrc/kernels/gemm_fp8.hip).

int8 keeps what is used element by element (``bias_act(bits=8)``, ``pack8``): its error is a fixed
fraction of the block's largest entry, 1/4 of e4m3's on normal data.

Sites of the reference model: hetseq/bert_modeling.py:104-116 (bias_gelu), :334-336, :383, :409, :419
(linear layers), :428-446 (checkpointed segments).
"""
import torch
from torch.autograd import forward_ad

from . import fused
from ._ext import C, use_kernels

BLOCK = 128
_DTYPES = (torch.float32, torch.bfloat16)


def _refuse_tangents(what, *ts):
    for t in ts:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError('{}: no forward-mode derivatives (an argument is a dual tensor)'.format(what))


def _check_act(x, what, tangents=False):
    if not torch.is_tensor(x) or x.dtype not in _DTYPES:
        raise TypeError('{}: an fp32 or bf16 tensor, got {}'.format(what, getattr(x, 'dtype', type(x).__name__)))
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('{}: needs a last dimension of at least 1, got shape {}'.format(what, tuple(x.shape)))
    if not tangents:
        _refuse_tangents(what, x)


def _check_weight(W, what):
    _check_act(W, what)
    if W.dim() != 2 or W.shape[0] < 1:
        raise ValueError('{}: a non-empty [out, in] weight, got shape {}'.format(what, tuple(W.shape)))


def _check_bias(b, n, like, what):
    if b is None:
        return
    if b.dtype != torch.float32 or tuple(b.shape) != (n,) or b.device != like.device:
        raise ValueError('{}: the bias must be fp32 [{}] on {}, got {} {} on {}'.format(
            what, n, like.device, b.dtype, tuple(b.shape), b.device))
    _refuse_tangents(what, b)


def _backward_checks(what, dy):
    if torch.is_grad_enabled():
        raise RuntimeError('{}: first derivatives only (create_graph=True is not supported)'.format(what))
    if use_kernels(dy):
        C().refuse_stale_leaves(dy, what)   # (captures only)


# ---------------------------------------------------------------- references (CPU, and the numerics oracle)
def _blocks_ref(x, largest):
    """x / 2^e per block of the last dimension, and 2^e, as [..., blocks, 128] fp32."""
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    a = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1, keepdim=True)
    m, e = torch.frexp(a)   # a = m 2^e, m in [1/2, 1)
    mt, et = torch.frexp(torch.tensor(float(largest)))
    e = torch.where(a > 0, e - int(et) + (m > float(mt)).to(e.dtype), torch.zeros_like(e)).clamp(min=-126)
    s = ((e + 127) << 23).view(torch.float32)
    return x * ((127 - e) << 23).view(torch.float32), s


def e4m3_ref(x):
    """The values of x's e4m3 codes (blocks along the last dimension), fp32."""
    v, s = _blocks_ref(x, 448.0)
    q = torch.where(torch.isfinite(v), v, torch.zeros_like(v)).to(torch.float8_e4m3fn).float()
    return torch.where(torch.isfinite(v), q * s, torch.full_like(v, float('nan'))).flatten(-2)[..., :x.shape[-1]]


def int8_ref(x):
    """The values of x's int8 codes (blocks along the last dimension), fp32."""
    v, s = _blocks_ref(x, 127.0)
    return torch.where(torch.isfinite(v), torch.round(v) * s, torch.full_like(v, float('nan'))).flatten(-2)[..., :x.shape[-1]]


def _gelu_grad_ref(u):
    c = 1.41421
    return 0.5 * (1.0 + torch.erf(u / c)) + u * torch.exp(-(u / c) ** 2) / (c * 3.141592653589793 ** 0.5)


# ---------------------------------------------------------------- operands
class Fp8Weight(object):
    """A weight's e4m3 codes for ``linear_fp8``: of W [N, K] blocked along K (the forward) and of W^T
    blocked along N (the data gradient; ``grad=False`` leaves it out: inference).  They are of W's
    values when it was built: a served model builds it once, training once per forward
    (``fp8_weights`` for a whole encoder)."""
    __slots__ = ('shape', 'dtype', 'device', 'q', 's', 'qt', 'st', 'ref')

    def __init__(self, W, grad=True):
        _check_weight(W, 'Fp8Weight')
        W = W.detach()
        self.shape, self.dtype, self.device = tuple(W.shape), W.dtype, W.device
        self.q = self.s = self.qt = self.st = self.ref = None
        if use_kernels(W):
            self.q, self.s, self.qt, self.st, _ = C().split8(_rows2(W), True, bool(grad))
        else:
            self.ref = (e4m3_ref(W), e4m3_ref(W.t()) if grad else None)

    @classmethod
    def _of(cls, W, q, s, qt, st):
        w = cls.__new__(cls)
        w.shape, w.dtype, w.device, w.ref = tuple(W.shape), W.dtype, W.device, None
        w.q, w.s, w.qt, w.st = q, s, qt, st
        return w

    @property
    def is_cuda(self):
        return self.device.type == 'cuda'

    def holds(self, other):
        """Whether this one's memory fits ``other``'s codes."""
        return (self.shape == other.shape and self.device == other.device and (self.ref is None) == (other.ref is None) and
                self.has_grad == other.has_grad)

    def assign(self, other):
        """``other``'s codes into this one's memory, which captured forwards read."""
        if self.ref is not None:
            self.ref = other.ref
            return
        with torch.inference_mode():   # (codes made in inference mode may be written in it only)
            for a, b in ((self.q, other.q), (self.s, other.s), (self.qt, other.qt), (self.st, other.st)):
                if a is not None:
                    a.copy_(b)

    @property
    def has_grad(self):
        return self.qt is not None or (self.ref is not None and self.ref[1] is not None)


def fp8_weights(Ws, grad=True):
    """``Fp8Weight`` of every weight in ``Ws`` (None stays None), contiguous fp32 ones on the GPU 64 to a
    launch: the ``codes`` of a whole encoder's layers."""
    out, batch = [None] * len(Ws), []
    for i, W in enumerate(Ws):
        if W is None:
            continue
        _refuse_tangents('fp8_weights', W)
        if use_kernels(W) and W.dim() == 2 and W.numel() and W.dtype == torch.float32 and W.is_contiguous() and W.data_ptr() % 16 == 0:
            batch.append(i)
        else:
            out[i] = Fp8Weight(W, grad)
    for o in range(0, len(batch), 64):
        part = batch[o:o + 64]
        for i, t in zip(part, C().split8_weights([Ws[j].detach() for j in part], bool(grad))):
            out[i] = Fp8Weight._of(Ws[i], *t)
    return out


def _check_codes(codes, shape, device, need_grad, what):
    if not isinstance(codes, Fp8Weight):
        raise TypeError('{}: codes must be an Fp8Weight, got {}'.format(what, type(codes).__name__))
    if codes.shape != shape or codes.device != device:
        raise ValueError('{}: codes of a {} weight on {}, the weight is {} on {}'.format(
            what, codes.shape, codes.device, shape, device))
    if (codes.ref is None) != use_kernels(codes):
        raise ValueError('{}: the Fp8Weight was built with the GPU kernels switched {}'.format(what, 'on' if codes.ref is None else 'off'))
    if need_grad and not codes.has_grad:
        raise ValueError('{}: x needs a gradient, the Fp8Weight was built with grad=False'.format(what))


def _rows2(x):
    """[.., K] as a 2-D operand with unit column stride (a contiguous copy if it has none)."""
    x2 = x.reshape(-1, x.shape[-1])
    ok = (x2.stride(1) == 1 or x2.shape[1] == 1) and (x2.stride(0) >= x2.shape[1] or x2.shape[0] <= 1)
    return x2 if ok else x2.contiguous()


# ---------------------------------------------------------------- linear
class _LinearFp8Fn(torch.autograd.Function):
    """One product over one weight, or over several stacked along the output features (Q / K / V).
    ``params``: the n weights (or none: frozen), then their n biases (or none).  ``bias``: the
    stacked bias added here; ``bgrad=False``: its gradient comes from the consumer."""

    @staticmethod
    def forward(ctx, x, w8, bias, mbox, bgrad, n, *params):
        N, K = w8.shape
        x2 = _rows2(x)
        ctx.wshape, ctx.mbox, ctx.xshape, ctx.n, ctx.bgrad = w8.shape, mbox, x.shape, n, bgrad
        ctx.Ws, ctx.bs = params[:n], params[n:]
        # the weight gradient reads the 8-bit copy of x blocked along the tokens
        keep = any(ctx.needs_input_grad[6:6 + n])
        if use_kernels(x):
            y, qt, st = C().linear_fp8_fwd(x2, w8.q, w8.s, bias, keep)
        else:
            y = e4m3_ref(x2) @ w8.ref[0].t()
            y = (y if bias is None else y + bias).to(x.dtype)
            qt, st = (e4m3_ref(x2.t()), None) if keep else (None, None)
        wt = (None, None)
        if ctx.needs_input_grad[0]:
            wt = (w8.qt, w8.st) if w8.ref is None else (w8.ref[1], None)
        ctx.save_for_backward(qt, st, *wt)
        return y.view(*x.shape[:-1], N)

    @staticmethod
    def backward(ctx, dy):
        _backward_checks('linear_fp8', dy)
        xt, xs, wt, ws = ctx.saved_tensors
        n, Ws, bs = ctx.n, ctx.Ws, ctx.bs
        N, K = ctx.wshape
        need_x = ctx.needs_input_grad[0]
        need_w = any(ctx.needs_input_grad[6:6 + n])
        need_b = ctx.bgrad and any(ctx.needs_input_grad[6 + n:])
        dy2 = _rows2(dy)
        M = dy2.shape[0]
        if not use_kernels(dy):
            dx = (e4m3_ref(dy2) @ wt.t()).to(dy.dtype).view(ctx.xshape) if need_x else None
            dW = e4m3_ref(dy2.t()) @ xt.t() if need_w else None
            db = dy2.float().sum(0) if need_b else None
            return (_residual(dx, ctx.mbox), None, None, None, None, None,
                    *_parts(dW, Ws, None), *_parts(db, bs, None))
        bslots, bview = _slots(bs) if need_b else (None, None)
        q, s, qt, st, db = C().split8(dy2, need_x, need_w and M > 0, need_b, bview)
        gW = _weight_grads(Ws, (N, K), qt, st, xt, xs, M) if need_w else (None,) * len(Ws)
        dx = _input_grad(q, s, wt, ws, N, M, ctx.xshape, dy.dtype == torch.bfloat16, ctx.mbox) if need_x else None
        return (dx, None, None, None, None, None, *gW, *_parts(db, bs, bslots, bview is not None))


def _weight_grads(Ws, shape, qt, st, xt, xs, M):
    """The stacked weights' gradients from the token-blocked codes of dy (qt, st) and of x (xt, xs): into
    their flat slots, on the side stream, where they have them."""
    slots, view = _slots(Ws)
    side = fused.side_begin(Ws[0].device, M) if view is not None and M > 0 else None
    with fused.side_ctx(side):
        if M == 0:
            dW = view.zero_() if view is not None else torch.zeros(shape, device=Ws[0].device)
        else:
            dW = C().gemm_fp8(qt, st, xt, xs, M, False, out=view)
        g = _parts(dW, Ws, slots, view is not None)
    fused._record(side, qt, st, xt, xs)
    return g


def _weight_grad(W, qt, st, xt, xs, M):
    return _weight_grads((W,), tuple(W.shape), qt, st, xt, xs, M)[0]


def _input_grad(q, s, wt, ws, N, M, xshape, bf16, mbox):
    """dx from the codes of dy (q, s) and of W^T (wt, ws), onto the residual gradient in ``mbox``."""
    acc = other = None
    if mbox is not None:
        acc, other = mbox.take(torch.bfloat16 if bf16 else torch.float32)
    acc = acc.view(M, xshape[-1]) if acc is not None else None
    dx = C().gemm_fp8(q, s, wt, ws, N, bf16, out=acc, beta=acc is not None).view(xshape)
    return dx if other is None else dx + other.view(xshape).to(dx.dtype)


def _slots(params):
    """The parameters' flat gradient slots and, if all have one and they lie back to back, the one
    view over them that a product writes directly."""
    slots = [fused.grad_slot(p) for p in params]
    if any(t is None for t in slots):
        return slots, None
    return slots, slots[0] if len(slots) == 1 else fused._adjacent_view(slots)


def _linear_nograd(x, w8, bias):
    """The product alone: nothing is kept for a backward.  (Inside ``apply`` a parameter counts as needing its
    gradient even under ``no_grad``.)"""
    if use_kernels(x):
        return C().linear_fp8_infer(x, w8.q, w8.s, w8.shape[1], bias)
    y = e4m3_ref(_rows2(x)) @ w8.ref[0].t()
    return (y if bias is None else y + bias).to(x.dtype).view(*x.shape[:-1], w8.shape[0])


def _parts(g, params, slots, direct=False):
    """The stacked gradient ``g`` as one gradient per parameter (in its slot, where it has one)."""
    if g is None:
        return (None,) * len(params)
    if direct:
        return tuple(slots)
    out, o = [], 0
    for i, p in enumerate(params):
        t = g[o:o + p.shape[0]].to(p.dtype)
        o += p.shape[0]
        if slots is not None and slots[i] is not None:
            t = slots[i].copy_(t)
        out.append(t)
    return tuple(out)


def _residual(dx, mbox):
    if mbox is None or dx is None:
        return dx
    g, other = mbox.take(dx.dtype)
    g = g if g is not None else other
    return dx if g is None else dx + g.view(dx.shape).to(dx.dtype)


def linear_fp8(x, W, b=None, res_grad=None, codes=None):
    """x W^T (+ b) with e4m3 operands (one power-of-two scale per block of 128; see the module's
    formulas).  ``x`` [.., K] fp32 or bf16 (the result has its type); ``W`` [N, K] a parameter, or an
    ``Fp8Weight`` (then it gets no gradient: inference, frozen layers); ``b`` fp32 [N].
    ``codes``: the parameter's ``Fp8Weight``, where the caller has made it for this forward
    (``fp8_weights``).  ``res_grad``: see ``ResidualGrad``.  First derivatives only; at most 2^22
    features in or out, fewer than 2^22 blocks of 128 x 128 of x, and in a training step 2^22 rows.
    Without gradients, few rows and a weight in 8 bits are one launch of exact products: a bf16 result may
    then be the other neighbour of the training forward's."""
    kept = isinstance(W, Fp8Weight)
    if kept and codes is None and torch.is_tensor(x) and use_kernels(x) and W.q is not None and not torch.is_grad_enabled():
        return C().linear_fp8_infer(x, W.q, W.s, W.shape[1], b)   # (checks its arguments as below)
    _check_act(x, 'linear_fp8')
    if not kept:
        _check_weight(W, 'linear_fp8')
    N, K = W.shape
    if x.shape[-1] != K:
        raise ValueError('linear_fp8: x has {} features, the weight takes {}'.format(x.shape[-1], K))
    if x.device != W.device:
        raise ValueError('linear_fp8: x on {}, the weight on {}'.format(x.device, W.device))
    _check_bias(b, N, x, 'linear_fp8')
    grad = torch.is_grad_enabled()
    if kept and codes is not None:
        raise ValueError('linear_fp8: codes go with a parameter; W is an Fp8Weight itself')
    w8 = W if kept else codes
    if w8 is not None:
        _check_codes(w8, (N, K), W.device, grad and x.requires_grad, 'linear_fp8')
    if use_kernels(x) and (not grad or res_grad is None and (kept or not _flat(W)) and not _flat(b)):
        # autograd keeps the gradients, or there are none: the whole layer is one node (bindings.cpp LinearFp8)
        return C().linear_fp8(x, None if kept else W, b, [] if w8 is None else [w8.q, w8.s, w8.qt, w8.st], grad)
    if w8 is None:
        w8 = Fp8Weight(W, grad and x.requires_grad)
    if not grad:
        return _linear_nograd(x, w8, b)
    if kept:
        return _LinearFp8Fn.apply(x, w8, b, res_grad, True, 0, *(() if b is None else (b,)))
    return _LinearFp8Fn.apply(x, w8, b, res_grad, True, 1, W, *(() if b is None else (b,)))


def _flat(p):
    return getattr(p, '_hx_flat', None) is not None


def linear3_fp8(x, wq, wk, wv, bq, bk, bv, res_grad=None, bias_grad=True, codes=None):
    """``linear3`` on e4m3 operands: the Q / K / V projections as one product (N = 3H).  ``codes``: the
    ``Fp8Weight`` of the three weights stacked."""
    _check_act(x, 'linear3_fp8')
    for W in (wq, wk, wv):
        _check_weight(W, 'linear3_fp8')
        if x.shape[-1] != W.shape[1] or x.device != W.device:
            raise ValueError('linear3_fp8: x {} on {}, a weight takes {} features on {}'.format(
                tuple(x.shape), x.device, W.shape[1], W.device))
    shape = (wq.shape[0] + wk.shape[0] + wv.shape[0], x.shape[-1])
    bs, bias = (), None
    if bq is not None:
        _refuse_tangents('linear3_fp8', bq, bk, bv)
        bs, bias = (bq, bk, bv), fused._adjacent_view([bq, bk, bv])
        bias = bias if bias is not None else torch.cat([t.detach() for t in bs], 0)
    _check_bias(bias, shape[0], x, 'linear3_fp8')
    need = torch.is_grad_enabled() and x.requires_grad
    if codes is not None:
        _check_codes(codes, shape, x.device, need, 'linear3_fp8')
    else:
        W = fused._adjacent_view([wq, wk, wv])
        codes = Fp8Weight(W if W is not None else torch.cat([wq.detach(), wk.detach(), wv.detach()], 0), need)
    if not torch.is_grad_enabled():
        return _linear_nograd(x, codes, bias)
    return _LinearFp8Fn.apply(x, codes, bias, res_grad, bool(bias_grad), 3, wq, wk, wv, *bs)


# ---------------------------------------------------------------- bias + GELU with an int8 checkpoint
def _bias_gelu_ref(y, b):
    return fused.gelu_ref(y.float() if b is None else y.float() + b).to(y.dtype)


class _BiasGelu8Fn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, b):
        ctx.b = b   # for its gradient slot; its values, which the slope is taken at, are saved: changed in place
        if use_kernels(y):   # before the backward they are an error
            out, q, s = C().gelu8_fwd(y, b, any(ctx.needs_input_grad))
            ctx.save_for_backward(q, s, b)
        else:
            out = _bias_gelu_ref(y, b)
            ctx.save_for_backward(int8_ref(y), None, b)
        return out

    @staticmethod
    def backward(ctx, dout):
        _backward_checks('bias_act(bits=8)', dout)
        q, s, b = ctx.saved_tensors
        need_b = ctx.needs_input_grad[1]
        if use_kernels(dout):
            dy, db = C().gelu8_bwd(dout.contiguous(), q, s, b, need_b, fused.grad_slot(ctx.b) if need_b else None)
            return dy, db
        dy = dout.float() * _gelu_grad_ref(q if b is None else q + b)
        return dy.to(dout.dtype), dy.reshape(-1, dy.shape[-1]).sum(0) if need_b else None


def bias_gelu8(y, b):
    """gelu(y + b); the backward reads y from int8 blocks (``bias_act(y, b, 'gelu', bits=8)``)."""
    _check_act(y, 'bias_act(bits=8)')
    _check_bias(b, y.shape[-1], y, 'bias_act(bits=8)')
    grad = torch.is_grad_enabled()
    if use_kernels(y) and not (grad and _flat(b)):
        return C().bias_gelu8(y, b)
    if not grad:
        return _bias_gelu_ref(y.contiguous(), b)
    return _BiasGelu8Fn.apply(y.contiguous(), b)


# ---------------------------------------------------------------- feed-forward
class _FfnFp8Fn(torch.autograd.Function):
    """gelu(x W1^T + b1) W2^T with the GELU's result and its input's gradient going straight to e4m3 codes
    (quant8.hip gelu8_split_k): neither tensor is written."""

    @staticmethod
    def products(x, c1, b1, c2, need_1, need_2, need_u):
        """The forward, and what the weight gradients (need_1, need_2) and whatever is behind the GELU (need_u) read."""
        x2, bf16 = _rows2(x), x.dtype == torch.bfloat16
        q, s, xt, xs, _ = C().split8(x2, True, need_1)
        y = C().gemm_fp8(q, s, c1.q, c1.s, c1.shape[1], bf16)
        q, s, *kept = C().gelu8_split_fwd(y, b1, need_2, need_u)
        out = C().gemm_fp8(q, s, c2.q, c2.s, c2.shape[1], bf16)
        return (out.view(*x.shape[:-1], c2.shape[0]), xt, xs, *kept)

    @staticmethod
    def forward(ctx, x, c1, c2, mbox, W1, b1, W2):
        need_x, _, _, _, need_1, need_b, need_2 = ctx.needs_input_grad
        ctx.xshape, ctx.mbox, ctx.W1, ctx.b1, ctx.W2 = x.shape, mbox, W1, b1, W2
        ctx.need_u = need_u = need_x or need_1 or need_b   # anything behind the GELU
        out, xt, xs, at, as_, kq, ks = _FfnFp8Fn.products(x, c1, b1, c2, need_1, need_2, need_u)
        w1 = (c1.qt, c1.st) if need_x else (None, None)
        w2 = (c2.qt, c2.st) if need_u else (None, None)
        ctx.save_for_backward(xt, xs, at, as_, kq, ks, *w1, *w2, b1)   # (b1: the slope is taken at its values)
        return out

    @staticmethod
    def backward(ctx, dy):
        _backward_checks('ffn_fp8', dy)
        xt, xs, at, as_, kq, ks, w1, w1s, w2, w2s, b1 = ctx.saved_tensors
        need_x, _, _, _, need_1, need_b, need_2 = ctx.needs_input_grad
        W1, W2 = ctx.W1, ctx.W2
        dy2, bf16 = _rows2(dy), dy.dtype == torch.bfloat16
        M = dy2.shape[0]
        q, s, qt, st, _ = C().split8(dy2, ctx.need_u, need_2 and M > 0)
        g2 = _weight_grad(W2, qt, st, at, as_, M) if need_2 else None
        dx = g1 = db = None
        if ctx.need_u:
            da = C().gemm_fp8(q, s, w2, w2s, W2.shape[0], bf16)
            q, s, qt, st, db = C().gelu8_split_bwd(da, kq, ks, b1, need_x, need_1 and M > 0, need_b,
                                                   fused.grad_slot(ctx.b1) if need_b else None)
            g1 = _weight_grad(W1, qt, st, xt, xs, M) if need_1 else None
            if need_x:
                dx = _input_grad(q, s, w1, w1s, W1.shape[0], M, ctx.xshape, bf16, ctx.mbox)
        return dx, None, None, None, g1, db, g2


def ffn_fp8(x, W1, b1, W2, res_grad=None, codes=(None, None)):
    """gelu(x W1^T + b1) W2^T on e4m3 operands: ``linear_fp8(bias_act(linear_fp8(x, W1), b1, 'gelu', bits=8),
    W2)`` -- the same roundings, b1's gradient summed in another order -- without writing the GELU's result
    or the gradient of its input.  ``W1`` [F, K], ``b1`` fp32 [F] or None, ``W2`` [N, F]; ``codes``: the ``Fp8Weight``
    of each where the caller has made it for this forward; ``res_grad`` as in ``linear_fp8``."""
    _check_act(x, 'ffn_fp8')
    for W in (W1, W2):
        _check_weight(W, 'ffn_fp8')
    if x.shape[-1] != W1.shape[1] or W2.shape[1] != W1.shape[0]:
        raise ValueError('ffn_fp8: x {}, weights {} and {}'.format(tuple(x.shape), tuple(W1.shape), tuple(W2.shape)))
    if x.device != W1.device or x.device != W2.device:
        raise ValueError('ffn_fp8: x on {}, the weights on {} and {}'.format(x.device, W1.device, W2.device))
    _check_bias(b1, W1.shape[0], x, 'ffn_fp8')
    if not use_kernels(x):
        return linear_fp8(bias_gelu8(linear_fp8(x, W1, res_grad=res_grad, codes=codes[0]), b1), W2, codes=codes[1])
    grad = torch.is_grad_enabled()
    need_x = grad and x.requires_grad
    need_u = need_x or grad and (W1.requires_grad or b1 is not None and b1.requires_grad)
    c = []
    for W, given, need in ((W1, codes[0], need_x), (W2, codes[1], need_u)):
        if given is not None:
            _check_codes(given, tuple(W.shape), W.device, need, 'ffn_fp8')
        c.append(given if given is not None else Fp8Weight(W, need))
    if not grad:   # (see _linear_nograd)
        return _FfnFp8Fn.products(x, c[0], b1, c[1], False, False, False)[0]
    return _FfnFp8Fn.apply(x, c[0], c[1], res_grad, W1, b1, W2)


# ---------------------------------------------------------------- kept activations
class Packed8(object):
    """A tensor kept as int8 blocks (``pack8``): codes [rows, blocks, 128], scale bytes [rows, blocks]."""
    __slots__ = ('q', 's', 'shape', 'dtype')

    def __init__(self, q, s, shape, dtype):
        self.q, self.s, self.shape, self.dtype = q, s, tuple(shape), dtype

    @property
    def nbytes(self):
        return self.q.numel() * self.q.element_size() + (self.s.numel() if self.s is not None else 0)


def pack8(x):
    """``x`` (fp32 or bf16) as int8 blocks along its last dimension: 1 + 1/128 bytes per element.  The blocks are
    values: no gradient flows back through ``unpack8(pack8(x))`` (``checkpoint8`` passes one through)."""
    _check_act(x, 'pack8')
    q, s = C().pack8(x) if use_kernels(x) else _pack8_ref(x.detach())
    return Packed8(q, s, x.shape, x.dtype)


def _pack8_ref(x):
    v, s = _blocks_ref(x.reshape(-1, x.shape[-1]), 127.0)
    q = torch.where(torch.isfinite(v), torch.round(v), torch.full_like(v, -128.0))
    return q.to(torch.int8).view(torch.uint8), (s.view(torch.int32) >> 23).to(torch.uint8).squeeze(-1)


def unpack8(p):
    """The values of a ``Packed8``, in its tensor's shape and type."""
    if not isinstance(p, Packed8):
        raise TypeError('unpack8: a Packed8 (ops.pack8), got {}'.format(type(p).__name__))
    if use_kernels(p.q):
        return C().unpack8(p.q, p.s, p.shape, p.dtype == torch.bfloat16)
    c = p.q.view(torch.int8).float()
    v = c * (p.s.to(torch.int32) << 23).view(torch.float32).unsqueeze(-1)
    v = torch.where(c == -128, torch.full_like(v, float('nan')), v)
    return v.flatten(-2)[..., :p.shape[-1]].to(p.dtype).view(p.shape)


class _Anchor(torch.autograd.Function):
    """A stand-in for x in the graph: its shape, type and gradient, one element of storage."""

    @staticmethod
    def forward(ctx, x):
        return x.new_zeros(()).expand(x.shape)

    @staticmethod
    def backward(ctx, g):
        return g


class _Restore8(torch.autograd.Function):
    """x while the segment first runs, its decoded 8-bit copy when it is recomputed."""

    @staticmethod
    def forward(ctx, anchor, box):
        return box.x.view_as(box.x) if box.x is not None else unpack8(box.kept)

    @staticmethod
    def backward(ctx, g):
        return g, None


class _Box(object):
    __slots__ = ('x', 'kept')


def checkpoint8(fn, x, *rest):
    """``fn(x, *rest)`` keeping only ``x`` in 8 bits (``pack8``) and ``rest`` as it is: the forward runs
    on ``x`` itself; the backward recomputes the segment from the decoded copy and passes x's
    gradient straight through the rounding.  ``fn`` returns a tensor or a tuple of them."""
    _check_act(x, 'checkpoint8', tangents=not torch.is_grad_enabled())
    if not torch.is_grad_enabled():
        return fn(x, *rest)
    from torch.utils.checkpoint import checkpoint
    box = _Box()
    box.x, box.kept = x.detach(), pack8(x)
    try:
        return checkpoint(lambda anchor, *r: fn(_Restore8.apply(anchor, box), *r), _Anchor.apply(x), *rest,
                          use_reentrant=False)
    finally:
        box.x = None
