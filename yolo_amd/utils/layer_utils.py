# coding: utf-8
"""conv2d / darknet53_body / yolo_block / upsample_layer with the signatures of reference
yolo_v3/utils/layer_utils.py, one HIP launch per call (yolo_conv_forward / yolo_upsample2x).

TF creates a layer's variables when the layer function is called; here the variables already exist
(a Darknet weight stream), so the calls consume them in creation order from the active
`variable_scope(params)` - the eager counterpart of `tf.variable_scope` + `Saver.restore`.
`yolov3.forward` does not go through these functions: it runs the whole fused plan
(yolo_net_forward).  These exist for layer-level drop-in use and tests.

`linear`, `qk_norm_rope` and `cross_attention` are the layers of a head in which cells, object queries or class prompts
attend to the feature maps; the reference has none.  Their weights are tensors the caller keeps, and unlike the layers above
they take and return bfloat16 as well as float32, without a cast at the boundary.
"""
from __future__ import division, print_function

import contextlib
import ctypes
import functools

import numpy as np
import torch
from torch.autograd import forward_ad

from .. import _lib, _tensor

_SCOPE = None


class _Scope(object):
    def __init__(self, params, dtype):
        self.params, self.dtype, self.next = list(params), dtype, 0
        self.handles = {}

    def take(self, cin, filters, kernel_size, strides):
        if self.next >= len(self.params):
            raise RuntimeError("variable_scope exhausted: more conv2d calls than weight sets")
        i, p = self.next, self.params[self.next]
        self.next += 1
        w = p["w"]
        if w.shape != (kernel_size, kernel_size, cin, filters):
            raise ValueError("conv #%d: weights %s do not fit conv2d(%d->%d, k=%d)" % (i, w.shape, cin, filters, kernel_size))
        if i not in self.handles:
            L = _lib.lib()
            h = ctypes.c_void_p()
            bn = "gamma" in p
            ps = [p["beta"], p["gamma"], p["mean"], p["var"]] if bn else [p["bias"], None, None, None]
            ps = [None if a is None else np.ascontiguousarray(a, np.float32) for a in ps]
            w = np.ascontiguousarray(w, np.float32)
            _lib.check(L.yolo_conv_create(_lib.DTYPES[self.dtype], cin, filters, kernel_size, strides, int(bn), w.ctypes.data,
                                          *[None if a is None else a.ctypes.data for a in ps], ctypes.byref(h)))
            self.handles[i] = h
        return self.handles[i]

    def close(self):
        for h in self.handles.values():
            _lib.lib().yolo_conv_destroy(h)
        self.handles = {}


@contextlib.contextmanager
def variable_scope(params, dtype="fp32"):
    """params: list of per-conv dicts in creation order (yolo_amd.weights.split_stream)."""
    global _SCOPE
    prev, _SCOPE = _SCOPE, _Scope(params, dtype)
    try:
        yield _SCOPE
    finally:
        _SCOPE.close()
        _SCOPE = prev


def conv2d(inputs, filters, kernel_size, strides=1, _residual=None):
    """layer_utils.py:9-21 (+ the arg_scope of model.py:32-36).  `_residual` fuses `net + shortcut`."""
    if _SCOPE is None:
        raise RuntimeError("conv2d must be called inside `with variable_scope(params):`")
    x = _tensor.as_dev_f32(inputs)
    B, H, W, cin = [int(v) for v in x.shape]
    h = _SCOPE.take(cin, filters, kernel_size, strides)
    L = _lib.lib()
    ho, wo = (H // strides, W // strides)
    out = _tensor.empty((B, ho, wo, filters))
    ws = _tensor.workspace(L.yolo_conv_workspace_bytes(h, B, H, W))
    res = _tensor.as_dev_f32(_residual) if _residual is not None else None
    _lib.check(L.yolo_conv_forward(h, x.data_ptr(), B, H, W, _tensor.ptr(res), out.data_ptr(), ws.data_ptr(), ws.numel(),
                                   _tensor.stream_ptr()))
    return out


def darknet53_body(inputs):
    """layer_utils.py:23-54 -> route_1, route_2, route_3."""
    def res_block(inputs, filters):
        shortcut = inputs
        net = conv2d(inputs, filters * 1, 1)
        return conv2d(net, filters * 2, 3, _residual=shortcut)        # net + shortcut fused (:28)

    net = conv2d(inputs, 32, 3, strides=1)
    net = conv2d(net, 64, 3, strides=2)
    net = res_block(net, 32)
    net = conv2d(net, 128, 3, strides=2)
    for i in range(2):
        net = res_block(net, 64)
    net = conv2d(net, 256, 3, strides=2)
    for i in range(8):
        net = res_block(net, 128)
    route_1 = net
    net = conv2d(net, 512, 3, strides=2)
    for i in range(8):
        net = res_block(net, 256)
    route_2 = net
    net = conv2d(net, 1024, 3, strides=2)
    for i in range(4):
        net = res_block(net, 512)
    route_3 = net
    return route_1, route_2, route_3


def yolo_block(inputs, filters):
    """layer_utils.py:56-65 -> (route, net)."""
    net = conv2d(inputs, filters * 1, 1)
    net = conv2d(net, filters * 2, 3)
    net = conv2d(net, filters * 1, 1)
    net = conv2d(net, filters * 2, 3)
    net = conv2d(net, filters * 1, 1)
    route = net
    net = conv2d(net, filters * 2, 3)
    return route, net


def upsample_layer(inputs, out_shape):
    """layer_utils.py:67-72: tf.image.resize_nearest_neighbor(inputs, (out_shape[1], out_shape[2]), align_corners=True).
    The exact-2x case of the network (where the TF rule equals src = dst // 2) runs the 16-byte-per-lane
    kernel; any other size the general one (TF 1.x rounding: src = min(round(dst * (in - 1) / (out - 1)), in - 1))."""
    x = _tensor.as_dev_f32(inputs)
    B, H, W, C = [int(v) for v in x.shape]
    new_height, new_width = int(out_shape[1]), int(out_shape[2])
    if new_height <= 0 or new_width <= 0:
        raise ValueError("upsample_layer: bad output size %dx%d" % (new_height, new_width))
    out = _tensor.empty((B, new_height, new_width, C))
    if new_height == 2 * H and new_width == 2 * W and C % 4 == 0:
        _lib.check(_lib.lib().yolo_upsample2x(x.data_ptr(), B, H, W, C, out.data_ptr(), _tensor.stream_ptr()))
    else:
        _lib.check(_lib.lib().yolo_upsample_nearest(x.data_ptr(), B, H, W, C, new_height, new_width, out.data_ptr(),
                                                    _tensor.stream_ptr()))
    return out


# ---- layers over feature maps without a counterpart in the reference -------------------------------------------------------
_DTYPE_CODES = {torch.float32: _lib.YOLO_DTYPE_F32, torch.bfloat16: _lib.YOLO_DTYPE_BF16}
_ACTIVATIONS = {None: 0, "linear": 0, "leaky": 1, "relu": 2, "gelu": 3, "silu": 4}


_Strides = ctypes.c_int64 * 3
_BF16 = torch.bfloat16
_INT_MAX = 0x7fffffff


def _no_tangents(**operands):
    """Forward-mode dual tensors would come out without their tangents.  Called inside a level of forward_ad only: looking at an operand
    costs 0.3 us."""
    for name, x in operands.items():
        if isinstance(x, torch.Tensor) and forward_ad.unpack_dual(x).tangent is not None:
            raise ValueError("%s has a tangent: yolo_amd implements the inference path only (no forward-mode derivatives)" % name)


def _dev(x, name, dev, dtype=None):
    """numpy / torch (any device) -> tensor of its own type (or `dtype`) on the current GPU `dev`, strides kept."""
    if not isinstance(x, torch.Tensor):
        x = torch.from_numpy(np.asarray(x))
        if x.dtype == torch.float64 and dtype is None:
            x = x.float()
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("%s requires a gradient: yolo_amd implements the inference path only (call under torch.no_grad())" % name)
    if x.dtype is not _BF16 and x.is_neg():                           # imaginary part of a conjugate: memory holds the negatives
        x = x.resolve_neg()
    if dtype is not None and x.dtype != dtype:
        x = x.to(dtype)
    if x.get_device() != dev:
        x = x.to(_tensor.device())
    return x


def _code(x, name):
    code = _DTYPE_CODES.get(x.dtype)
    if code is None:
        raise ValueError("%s must be float32 or bfloat16, got %s" % (name, x.dtype))
    return code


def _same_type(x, like, name):
    if x.dtype != like.dtype:
        raise ValueError("%s is %s, expected %s" % (name, x.dtype, like.dtype))
    return x


def _param(x, n, name, dev):
    """Bias / norm weight: [n] contiguous, float32 or bfloat16 -> (tensor or None, type code)."""
    if x is None:
        return None, 0
    x = _dev(x, name, dev)
    if x.shape != (n,):
        raise ValueError("%s must be [%d], got %s" % (name, n, tuple(x.shape)))
    return x.contiguous(), _code(x, name)


def _fits(name, *sizes):
    """The C entries take int sizes, and ctypes would pass on the low 32 bits of a longer one.  Called for tensors of 2^31 elements and more."""
    if max(sizes) > _INT_MAX:
        raise ValueError("%s: sizes %s, each must be below 2^31" % (name, sizes))


def _gpu():
    """Index of the current GPU; like `_tensor.device()` an error without one."""
    try:
        return torch.cuda.current_device()
    except Exception:
        _tensor.device()
        raise


def _rows(x):
    """[..., n] -> (tensor, elements between rows) with all leading dimensions as rows of one stride; copied if there is none."""
    n = x.shape[-1]
    if x.is_contiguous():
        return x, n
    if x.dim() == 1:
        return x.contiguous(), n
    st, sh = x.stride(), x.shape
    ok = n == 1 or st[-1] == 1
    rows, ld = 1, None                                                # innermost row dimension of more than one row sets the stride
    for i in range(x.dim() - 2, -1, -1):
        if sh[i] == 1:
            continue
        if ld is None:
            ld = st[i]
        ok = ok and st[i] == rows * ld
        rows *= sh[i]
    if ok and (ld is None or ld >= n):
        return x, n if ld is None else ld
    return x.contiguous(), n


def linear(inputs, weight, bias=None, activation=None, residual=None):
    """act(inputs @ weight.T + bias) + residual in one launch: inputs [..., K] (a map's cells [B, H, W, K] as they are), weight
    [N, K], bias [N], residual [..., N] -> [..., N], float32 or bfloat16 throughout (bias: either).  activation: None, "leaky"
    (slope 0.1), "relu", "gelu" (error function) or "silu"; the residual is added after it, as in res_block.  yolo_linear."""
    if forward_ad._current_level >= 0:
        _no_tangents(inputs=inputs, weight=weight, bias=bias, residual=residual)
    dev = _gpu()
    x, w = _dev(inputs, "inputs", dev), _dev(weight, "weight", dev)
    code = _code(x, "inputs")
    _same_type(w, x, "weight")
    act = _ACTIVATIONS.get(activation, -1)
    if act < 0:
        raise ValueError("linear: unknown activation %r" % (activation,))
    shape, wshape = tuple(x.shape), w.shape
    if not shape or len(wshape) != 2 or wshape[1] != shape[-1] or wshape[1] == 0 or wshape[0] == 0:
        raise ValueError("linear: inputs %s do not fit weight %s" % (shape, tuple(wshape)))
    N, K = wshape
    if w.numel() > _INT_MAX:
        _fits("linear", N, K)
    b, bcode = _param(bias, N, "bias", dev)
    shape = shape[:-1] + (N,)
    r, r_ld = None, 0
    if residual is not None:
        r = _same_type(_dev(residual, "residual", dev), x, "residual")
        if r.shape != shape:
            raise ValueError("linear: residual %s, expected %s" % (tuple(r.shape), shape))
        r, r_ld = _rows(r)
    out = x.new_empty(shape)
    x, x_ld = _rows(x)
    w, w_ld = _rows(w)
    _lib.check(_lib.lib().yolo_linear(code, x.data_ptr(), x_ld, w.data_ptr(), w_ld, _tensor.ptr(b), bcode, _tensor.ptr(r), r_ld,
                                      out.data_ptr(), N, out.numel() // N, N, K, act, _tensor.stream_ptr(dev)))
    return out


def rope_frequencies(rotary_dim, base=10000.0, axes=1):
    """float64 [rotary_dim / 2] on the current GPU, radians per position of every pair of `qk_norm_rope`: base ** (-i / n) for the
    n = rotary_dim / 2 / axes pairs of an axis, the axes one after the other."""
    if axes not in (1, 2) or rotary_dim <= 0 or rotary_dim % (2 * axes):
        raise ValueError("rope_frequencies: rotary_dim %r does not split into pairs over %r axes" % (rotary_dim, axes))
    n = rotary_dim // 2 // axes
    f = float(base) ** (-np.arange(n, dtype=np.float64) / n)
    return torch.from_numpy(np.tile(f, axes)).to(_tensor.device())


def _heads(x, name):
    """[B, L, H, D] with a contiguous last dimension -> (tensor, ctypes strides of batch, token, head)."""
    if x.dim() != 4:
        raise ValueError("%s must be [B, L, H, D], got %s" % (name, tuple(x.shape)))
    if x.numel() > _INT_MAX:
        _fits(name, *x.shape)
    st = x.stride()
    if st[3] != 1 and x.shape[3] > 1:
        x = x.contiguous()
        st = x.stride()
    return x, _Strides(st[0], st[1], st[2])


def _attention_operand(x, D):
    """[B, L, H, D] -> (tensor, ctypes strides of batch, token, head); copied if D is not contiguous or, where the matrix-core kernels
    could run (D a multiple of 8), if a row does not start on 16 bytes."""
    st = x.stride()
    if (st[3] != 1 and D > 1) or (D % 8 == 0 and (x.data_ptr() | (st[0] | st[1] | st[2]) * x.element_size()) & 15):
        x = x.clone(memory_format=torch.contiguous_format)
        st = x.stride()
    return x, _Strides(st[0], st[1], st[2])


def _positions(p, B, L, axes, name):
    """Tensor on the GPU -> (contiguous tensor, batched).  [L] / [B, L] for one axis, [L, 2] / [B, L, 2] for two; a trailing 1 is allowed for one."""
    if p.dtype not in (torch.int32, torch.int64):
        raise ValueError("%s must be int32 or int64, got %s" % (name, p.dtype))
    shape = tuple(p.shape)
    tail = () if axes == 1 and (shape == (L,) or shape == (B, L)) else (axes,)
    if shape == (L,) + tail:
        return p.contiguous(), 0
    if shape == (B, L) + tail:
        return p.contiguous(), 1
    raise ValueError("%s %s fits neither %s nor %s" % (name, shape, (L,) + tail, (B, L) + tail))


def qk_norm_rope(q, k, q_weight=None, k_weight=None, frequencies=None, q_positions=None, k_positions=None, eps=1e-6,
                 interleaved=False, axes=None):
    """Root-mean-square norm of every head of the queries and keys, then the rotation by position, in one launch:
    q [B, Lq, Hq, D], k [B, Lk, Hk, D] (any strides over a contiguous D; None: queries only) -> new packed tensors (q, k).
    *_weight [D] or None (ones).  frequencies: float64 [rotary_dim / 2] of `rope_frequencies` (None: no rotation); elements past
    rotary_dim are normalised only.  Positions int32 / int64: [L] or [B, L]; for the cells of a map [L, 2] or [B, L, 2] (row,
    column), where the first half of the pairs turns by the row and the second by the column.  `axes` (1 or 2) says which where
    None would leave [B, L] = [L, 2] open.  Pairs are (i, i + rotary_dim / 2), or (2i, 2i + 1) if `interleaved`.
    yolo_qk_norm_rope."""
    if forward_ad._current_level >= 0:
        _no_tangents(q=q, k=k, q_weight=q_weight, k_weight=k_weight, frequencies=frequencies)
    dev = _gpu()
    q, qs = _heads(_dev(q, "q", dev), "q")
    code = _code(q, "q")
    B, Lq, Hq, D = q.shape
    Lk, Hk, ks, ko = 0, 0, None, None
    if k is not None:
        k, ks = _heads(_same_type(_dev(k, "k", dev), q, "k"), "k")
        Lk, Hk = k.shape[1:3]
        if k.shape[0] != B or k.shape[3] != D:
            raise ValueError("qk_norm_rope: k %s does not fit q %s" % (tuple(k.shape), tuple(q.shape)))
        ko = q.new_empty((B, Lk, Hk, D))
    qw, qwc = _param(q_weight, D, "q_weight", dev)
    kw, kwc = _param(k_weight if k is not None else None, D, "k_weight", dev)
    if qw is not None and kw is not None and qwc != kwc:
        raise ValueError("q_weight and k_weight must be of one type")
    qp = kp = None
    R, pos64, qb, kb = 0, 0, 0, 0
    if frequencies is not None:
        frequencies = _dev(frequencies, "frequencies", dev, torch.float64).contiguous()
        if frequencies.dim() != 1 or not 0 < 2 * frequencies.shape[0] <= D:
            raise ValueError("qk_norm_rope: frequencies %s for heads of %d" % (tuple(frequencies.shape), D))
        R = 2 * int(frequencies.shape[0])
        if q_positions is None or (k is not None and k_positions is None):
            raise ValueError("qk_norm_rope: frequencies need positions")
        q_positions = _dev(q_positions, "q_positions", dev)
        if axes is None:
            if tuple(q_positions.shape) == (2, 2) == (B, Lq):
                raise ValueError("qk_norm_rope: positions [2, 2] of 2 x 2 queries may be one axis or two: pass axes")
            axes = 2 if q_positions.dim() > 1 and q_positions.shape[-1] == 2 and tuple(q_positions.shape) != (B, Lq) else 1
        if axes not in (1, 2) or R // 2 % axes:
            raise ValueError("qk_norm_rope: %d pairs over %r axes" % (R // 2, axes))
        qp, qb = _positions(q_positions, B, Lq, axes, "q_positions")
        if k is not None:
            kp, kb = _positions(_dev(k_positions, "k_positions", dev), B, Lk, axes, "k_positions")
            if kp.dtype != qp.dtype:
                kp, qp = kp.long(), qp.long()
        pos64 = int(qp.dtype == torch.int64)
    qo = q.new_empty((B, Lq, Hq, D))
    if D == 0 or Hq == 0 or (k is not None and Hk == 0):
        raise ValueError("qk_norm_rope: no heads in q %s" % (tuple(q.shape),))
    _lib.check(_lib.lib().yolo_qk_norm_rope(
        code, B, D, q.data_ptr(), qs, Lq, Hq, _tensor.ptr(qw), _tensor.ptr(qp), qo.data_ptr(),
        _tensor.ptr(k), ks, Lk, Hk, _tensor.ptr(kw), _tensor.ptr(kp), _tensor.ptr(ko), qwc if qw is not None else kwc,
        _tensor.ptr(frequencies), R, axes or 1, pos64, qb, kb, int(bool(interleaved)), float(eps), _tensor.stream_ptr(dev)))
    return qo, ko


@functools.lru_cache(maxsize=4096)
def _attention_workspace(*sizes):
    return _lib.lib().yolo_cross_attention_workspace_bytes(*sizes)


def cross_attention(q, k, v, key_lens=None, key_mask=None, scale=None):
    """softmax(scale * q k^T) v: q [B, Lq, Hq, D] over the states k, v [B, Lk, Hk, D] of another length (any strides over a
    contiguous D, so the halves of one key / value projection go in as views); Hq a multiple of Hk, query head h reads key head
    h // (Hq // Hk).  key_lens [B] int32: keys from key_lens[b] on are padding; key_mask [B, Lk] bool: False leaves a key out.
    What is left out has no influence whatever it holds; a row with no key left is zero. bfloat16 rounds the weights of the
    values where a key head serves more than 32 rows (queries times the query heads that share it).  scale: None = D ** -0.5.  D up to 256;
    tensors whose rows do not start on 16 bytes are copied first, head sizes that are not multiples of 8 padded.
    -> [B, Lq, Hq, D] packed.  yolo_cross_attention."""
    if forward_ad._current_level >= 0:
        _no_tangents(q=q, k=k, v=v)
    dev = _gpu()
    q = _dev(q, "q", dev)
    code = _code(q, "q")
    k, v = _same_type(_dev(k, "k", dev), q, "k"), _same_type(_dev(v, "v", dev), q, "v")
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("cross_attention: q %s and k %s must be [B, L, H, D]" % (tuple(q.shape), tuple(k.shape)))
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1:3]
    if q.numel() > _INT_MAX or k.numel() > _INT_MAX:
        _fits("cross_attention", B, Lq, Lk, Hq, Hk, D)
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError("cross_attention: q %s, k %s, v %s do not fit" % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if D == 0 or Hk == 0 or Hq == 0 or Hq % Hk:
        raise ValueError("cross_attention: %d query heads over %d key heads of %d" % (Hq, Hk, D))
    if scale is None:
        scale = D ** -0.5
    if D % 8 and D <= 256 and Lk:
        # zeros up to the next multiple of 8 change no score and add no result: copies, but on the matrix cores
        pad = (0, -D % 8)
        return cross_attention(*[torch.nn.functional.pad(x, pad) for x in (q, k, v)], key_lens, key_mask, scale)[..., :D].contiguous()
    (q, qs), (k, ks), (v, vs) = _attention_operand(q, D), _attention_operand(k, D), _attention_operand(v, D)
    if key_lens is not None:
        key_lens = _dev(key_lens, "key_lens", dev)
        if tuple(key_lens.shape) != (B,) or key_lens.dtype not in (torch.int32, torch.int64):
            raise ValueError("key_lens must be int32 [%d], got %s %s" % (B, key_lens.dtype, tuple(key_lens.shape)))
        if key_lens.dtype == torch.int64:
            key_lens = key_lens.clamp(0, Lk).to(torch.int32)
        key_lens = key_lens.contiguous()
    if key_mask is not None:
        key_mask = _dev(key_mask, "key_mask", dev)
        if tuple(key_mask.shape) != (B, Lk) or key_mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError("key_mask must be bool [%d, %d], got %s %s" % (B, Lk, key_mask.dtype, tuple(key_mask.shape)))
        key_mask = key_mask.contiguous()
    out = q.new_empty((B, Lq, Hq, D))
    L = _lib.lib()
    need = _attention_workspace(code, B, Lq, Lk, Hq, Hk, D)
    ws = q.new_empty((need,), dtype=torch.uint8) if need else None
    _lib.check(L.yolo_cross_attention(code, q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, _tensor.ptr(key_lens),
                                      _tensor.ptr(key_mask), B, Lq, Lk, Hq, Hk, D, float(scale),
                                      out.data_ptr(), _tensor.ptr(ws), need, _tensor.stream_ptr(dev)))
    return out
