"""linear, qk_norm_rope and cross_attention against plain implementations in float64 on the same (already rounded) inputs.

Tolerances, all derived before the first run.  u = finfo(type).eps / 2 is the largest relative error of one rounding.
 * linear: products of rounded inputs are summed in f32: |error| <= K * 2^-24 * sum|x w| in the worst order, plus bias and the
   activation (slope <= 1.13 for gelu and silu, formula within 2^-20 of the value's scale), plus one rounding of the result:
   |err| <= u |y| + 1.13 * (K + 8) * 2^-24 * (sum |x w| + |b|) + 2^-20 * |pre| + 2^-22 |r|.
 * qk_norm_rope: a handful of f32 operations on the two partners of a pair: |err| <= u |y| + 2^-20 * (|u_i| + |v_i|).  The sum
   of D <= 256 squares is off by at most 2^-16 relatively in the worst order, half of that in the square root: the bound takes 2^-16.
   The angle a is a product in float64 reduced by another: 2^-51 |a| between two ways to form it.
 * cross_attention: a score is off by ds <= (D + 4) 2^-24 sum|q k| scale, so a weight by a factor exp(2 ds) at most, and the sum of
   n weights by n 2^-24; in bf16 the weights are rounded once more, u each.  With P the exact weights and A = P |v|:
   |err| <= u |o| + (e^(2 ds) - 1 + 2 n 2^-24 + 2^-18 + (u if bf16)) * 2 A.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def L(torch_cuda):
    from yolo_amd.utils import layer_utils
    return layer_utils


def rand(shape, t, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(t).cuda()


def within(got, ref, bound, what):
    g, r, b = got.double().cpu(), ref.cpu(), bound.cpu()
    assert g.shape == r.shape, what
    assert torch.isfinite(g).all(), what
    over = (g - r).abs() - b
    assert float(over.max()) <= 0, "%s: %.3g over the bound at %s" % (what, float(over.max()), np.unravel_index(int(over.argmax()), over.shape))


# ---- linear ----------------------------------------------------------------------------------------------------------------
ACTS = {None: lambda y: y, "leaky": lambda y: torch.where(y > 0, y, 0.1 * y), "relu": lambda y: y.clamp(min=0),
        "gelu": lambda y: y * torch.special.ndtr(y), "silu": lambda y: y * torch.sigmoid(y)}


def check_linear(L, x, w, b, act, r, what):
    got = L.linear(x, w, b, activation=act, residual=r)
    x2, w2 = x.double().cpu().reshape(-1, x.shape[-1]), w.double().cpu()
    pre = x2 @ w2.t().contiguous()
    mag = x2.abs() @ w2.abs().t().contiguous()
    if b is not None:
        pre = pre + b.double().cpu()
        mag = mag + b.double().cpu().abs()
    y = ACTS[act](pre)
    u = torch.finfo(x.dtype).eps / 2
    bound = 1.13 * (x.shape[-1] + 8) * 2.0 ** -24 * mag + 2.0 ** -20 * pre.abs()
    if r is not None:
        r2 = r.double().cpu().reshape(y.shape)
        y = y + r2
        bound = bound + 2.0 ** -22 * r2.abs()
    bound = bound * (1 + u) + u * y.abs() + 1e-38
    assert got.dtype == x.dtype and got.is_contiguous()
    within(got.reshape(y.shape), y, bound, what)
    return got


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 8, 16), (1, 1024, 1024), (3, 7, 5), (16, 255, 85), (17, 64, 32), (31, 33, 129), (80, 512, 1000),
                                   (129, 72, 130), (700, 255, 255), (1001, 256, 512), (1300, 136, 1025), (4097, 40, 264), (2704, 1024, 256)])
@pytest.mark.parametrize("act,bias,res", [(None, False, False), ("leaky", True, True)])
def test_linear_sizes(L, t, m, k, n, act, bias, res):
    x, w = rand((m, k), t, 1), rand((n, k), t, 2, k ** -0.5)
    check_linear(L, x, w, rand((n,), t, 3) if bias else None, act, rand((m, n), t, 4) if res else None, (t, m, k, n))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("m,k,n", [(16833, 64, 32), (17000, 72, 31), (20001, 33, 17), (33000, 20, 1)])
@pytest.mark.parametrize("act,bias,res", [(None, False, False), ("silu", True, True)])
def test_linear_narrow_outputs(L, t, m, k, n, act, bias, res):
    x, w = rand((m, k), t, 1), rand((n, k), t, 2, k ** -0.5)
    check_linear(L, x, w, rand((n,), t, 3) if bias else None, act, rand((m, n), t, 4) if res else None, (t, m, k, n))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("m,n", [(20, 40), (300, 80), (1500, 300), (9000, 20), (4100, 1100)])
@pytest.mark.parametrize("k", [1, 3, 7, 9, 61, 65, 127, 263])
def test_linear_rows_that_end_inside_a_piece(L, t, m, n, k):
    """Unaligned rows inside a larger matrix of NaN: nothing outside a row has influence, wherever its last 16 bytes start."""
    big_x, big_w = torch.full((m, k + 7), float("nan"), dtype=t, device="cuda"), torch.full((n, k + 5), float("nan"), dtype=t, device="cuda")
    x, w = big_x[:, 3:3 + k], big_w[:, 2:2 + k]
    x.copy_(rand((m, k), t, 1))
    w.copy_(rand((n, k), t, 2, k ** -0.5))
    check_linear(L, x, w, rand((n,), t, 3), None, None, (t, m, k, n))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("m,k,n", [(12300, 64, 640), (12301, 136, 648), (12289, 72, 641), (2800, 512, 2056), (6001, 264, 1100), (1537, 200, 1030),
                                   (20000, 96, 96), (9500, 320, 130), (30000, 24, 250), (4160, 1000, 520)])
@pytest.mark.parametrize("act,bias,res", [(None, False, False), ("gelu", True, True)])
def test_linear_tile_shapes(L, t, m, k, n, act, bias, res):
    """Sizes on either side of every choice of a tile, whole and ragged in both directions."""
    x, w = rand((m, k), t, 1), rand((n, k), t, 2, k ** -0.5)
    check_linear(L, x, w, rand((n,), t, 3) if bias else None, act, rand((m, n), t, 4) if res else None, (t, m, k, n))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("m", [5, 2100])
def test_linear_activations(L, t, act, m):
    # pre-activations from the far negative tail to the far positive one
    x, w = rand((m, 64), t, 5), rand((512, 64), t, 6, 0.7)
    check_linear(L, x, w, rand((512,), F32, 7, 3.0), act, rand((m, 512), t, 8), (t, act, m))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("m", [9, 1500])
def test_linear_strides_and_alignment(L, t, m):
    big = rand((m, 3, 200), t, 9)
    wide = rand((300, 520), t, 10, 0.1)
    for x in (big[:, 1], big[:, 1, :64], big[:, 0, 1:66], big[:, 2, 3:100]):
        k = x.shape[-1]
        for w in (wide[:, :k], wide[:, 5:5 + k], wide[::2, :k], wide[1:60, 8:8 + k]):
            r = rand((m, 2, w.shape[0] + 3), t, 11)[:, 1, 1:w.shape[0] + 1]
            check_linear(L, x, w, rand((w.shape[0],), t, 12), "relu", r, (t, m, x.shape, x.stride(), w.shape, w.stride()))
    # transposed and broadcast operands, leading dimensions, one dimension, numpy
    xt = rand((64, m), t, 13).t()
    check_linear(L, xt, wide[:, :64], None, None, rand((1, 300), t, 14).expand(m, 300), (t, m, "transposed"))
    x4 = rand((2, m, 3, 64), t, 15)
    got = check_linear(L, x4, wide[:, :64], None, "silu", None, (t, m, "4d"))
    assert got.shape == (2, m, 3, 300)
    assert torch.equal(L.linear(x4.permute(1, 0, 2, 3), wide[:, :64], activation="silu"), got.permute(1, 0, 2, 3).contiguous())
    assert L.linear(x4[0, 0, 0], wide[:, :64]).shape == (300,)
    assert L.linear(x4[:0], wide[:, :64]).shape == (0, m, 3, 300)
    a = np.random.default_rng(0).random((4, 8), np.float32)
    check = L.linear(a, a)
    assert check.is_cuda and np.allclose(check.cpu().numpy(), a @ a.T, atol=1e-5)


def test_linear_infinities_stay_in_their_rows(L):
    for t, m in ((BF16, 40), (F32, 40), (BF16, 1600), (F32, 1600)):
        x, w = rand((m, 128), t, 16), rand((640, 128), t, 17)
        clean = L.linear(x, w)
        x2, w2 = x.clone(), w.clone()
        x2[7, 3] = float("inf")
        x2[11, 5] = float("nan")
        w2[13, 100] = float("nan")
        got = L.linear(x2, w2)
        keep = torch.ones_like(clean, dtype=torch.bool)
        keep[7] = keep[11] = False
        keep[:, 13] = False
        assert torch.equal(got[keep], clean[keep]) and not torch.isfinite(got[7]).any() and got[11].isnan().all() and got[:, 13].isnan().all()


def test_linear_leaves_the_surroundings(L):
    """Odd sizes through the C entry: nothing outside the [M, N] block of a wider buffer is written, nothing past K read into it."""
    from yolo_amd import _lib, _tensor
    for t, code in ((F32, 0), (BF16, 1)):
        for m, n, k, ld in ((5, 7, 9, 16), (300, 131, 40, 136), (1100, 1025, 24, 1032)):
            x = torch.full((m + 1, ld + 8), float("nan"), dtype=t, device="cuda")
            x[:m, :k] = rand((m, k), t, 18)
            w = torch.full((n, ld + 8), float("nan"), dtype=t, device="cuda")
            w[:, :k] = rand((n, k), t, 19)
            out = torch.full((m + 2, n + 5), 7.0, dtype=t, device="cuda")
            _lib.check(_lib.lib().yolo_linear(code, x.data_ptr(), ld + 8, w.data_ptr(), ld + 8, None, 0, None, 0, out[1:].data_ptr(), n + 5,
                                              m, n, k, 0, _tensor.stream_ptr()))
            ref = L.linear(x[:m, :k].contiguous(), w[:, :k].contiguous())
            assert torch.equal(out[1:m + 1, :n], ref)
            assert (out[0] == 7).all() and (out[m + 1] == 7).all() and (out[:, n:] == 7).all()


# ---- qk_norm_rope --------------------------------------------------------------------------------------------------------------
def ref_norm_rope(x, w, f, p, axes, interleaved, eps):
    """-> result, bound without the final rounding; float64 on the CPU.  p: [B, L, axes]."""
    h = x.double().cpu()
    h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    if w is not None:
        h = h * w.double().cpu()
    y, mag, turn = h.clone(), h.abs(), 0.0
    if f is not None:
        half = f.numel()
        axis = torch.arange(half) * axes // half
        a = p.double().cpu()[..., axis] * f.double().cpu()
        c, s = torch.cos(a)[:, :, None], torch.sin(a)[:, :, None]
        iu = torch.arange(half) * 2 if interleaved else torch.arange(half)
        iv = iu + (1 if interleaved else half)
        y[..., iu], y[..., iv] = h[..., iu] * c - h[..., iv] * s, h[..., iu] * s + h[..., iv] * c
        both = h[..., iu].abs() + h[..., iv].abs()
        mag[..., iu], mag[..., iv] = both, both
        turn = torch.zeros(h.shape[:2] + (1, h.shape[3]), dtype=torch.float64)
        turn[..., iu] = turn[..., iv] = (2.0 ** -51 * a.abs())[:, :, None]
    return y, (2.0 ** -16 + turn) * mag


def check_qk(L, q, k, qw, kw, f, qp, kp, axes=1, interleaved=False, eps=1e-6):
    qo, ko = L.qk_norm_rope(q, k, qw, kw, f, qp, kp, eps=eps, interleaved=interleaved, axes=axes)
    for x, w, p, o in ((q, qw, qp, qo), (k, kw, kp, ko)):
        if x is None:
            assert o is None
            continue
        if p is not None:
            p = p.reshape((-1, x.shape[1], axes)).expand(x.shape[0], -1, -1)
        y, bound = ref_norm_rope(x, w, f, p, axes, interleaved, eps)
        assert o.is_contiguous() and o.dtype == x.dtype
        within(o, y, bound + torch.finfo(x.dtype).eps / 2 * (y.abs() + bound) + 1e-38, (x.dtype, x.shape, axes, interleaved))
    return qo, ko


def grid_positions(n, batch, axes, start=0, dtype=torch.int32):
    p = torch.arange(n)[None, :, None] + start + torch.arange(batch)[:, None, None] * 3 + torch.arange(axes) * 7
    return p.to(dtype).cuda()


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axes", [1, 2])
@pytest.mark.parametrize("d", [4, 8, 20, 32, 64, 80, 96, 100, 128, 256])
def test_qk_head_sizes(L, t, interleaved, axes, d):
    q, k = rand((2, 13, 6, d), t, 20), rand((2, 40, 3, d), t, 21, 0.3)
    f = L.rope_frequencies(d, axes=axes)
    check_qk(L, q, k, rand((d,), t, 22), rand((d,), t, 23), f, grid_positions(13, 2, axes), grid_positions(40, 2, axes), axes, interleaved)


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("b,lq,lk,hq,hk", [(1, 1, 0, 1, 1), (1, 1, 1, 8, 8), (5, 1, 0, 32, 1), (3, 100, 2704, 8, 2), (1, 361, 7, 1, 40), (2, 169, 1444, 5, 3),
                                           (2, 3, 2, 300, 70)])
def test_qk_shapes(L, t, b, lq, lk, hq, hk):
    d = 64
    q = rand((b, lq, hq, d), t, 24)
    k = rand((b, lk, hk, d), t, 25) if lk else None
    f = L.rope_frequencies(d)
    qp = grid_positions(lq, 1, 1, 5)[0, :, 0]
    kp = grid_positions(lk, b, 1, 9)[..., 0] if lk else None
    check_qk(L, q, k, rand((d,), F32, 26), None, f, qp, kp)


def test_qk_strides_partial_rotation_and_absent_parts(L):
    for t in (BF16, F32):
        qkv = rand((2, 30, 3, 4, 64), t, 27)
        f = L.rope_frequencies(64)
        p = torch.arange(30, device="cuda")                                       # int64
        check_qk(L, qkv[:, :, 0], qkv[:, :, 1], None, None, f, p, p)
        check_qk(L, qkv[:, ::2, 0], qkv[:, 1::3, 2], None, None, f, p[:15], p[:10])
        odd = rand((2, 30, 4, 67), t, 28)[..., 1:65]                              # rows off 16-byte boundaries
        check_qk(L, odd, odd.transpose(1, 2), None, None, f, p, p[:4])
        w = rand((64,), t, 29)
        for r in (2, 16, 32, 62):                                                 # the rest of a head is normalised only
            for il in (False, True):
                check_qk(L, qkv[:, :, 0], None, w, None, L.rope_frequencies(r), p, None, interleaved=il)
        check_qk(L, qkv[:, :, 0], qkv[:, :, 1], w, w, None, None, None)           # norm alone
        assert L.qk_norm_rope(qkv[:, :0, 0], None)[0].shape == (2, 0, 4, 64)
        assert L.qk_norm_rope(qkv[:0, :, 0], qkv[:0, :, 1])[1].shape == (0, 30, 4, 64)


def test_qk_far_positions_zeros_and_large_values(L):
    f = L.rope_frequencies(128)
    for t in (BF16, F32):
        q = rand((1, 5, 2, 128), t, 30)
        q[0, 0] = 0
        q[0, 1] *= 1e15
        q[0, 2] *= 1e-12
        p = torch.tensor([0, 1, 1000003, 2 ** 31 - 1, -77], device="cuda")
        qo, _ = check_qk(L, q, None, None, None, f, p, None)
        assert (qo[0, 0] == 0).all()
        check_qk(L, q, None, None, None, f, p.to(torch.int32), None)
        check_qk(L, q[:, :1], None, None, None, f, torch.tensor([2 ** 40], device="cuda"), None)


# ---- cross_attention -----------------------------------------------------------------------------------------------------------
def kept_keys(b, lk, lens, mask):
    keep = torch.ones((b, lk), dtype=torch.bool)
    if lens is not None:
        keep &= torch.arange(lk)[None, :] < lens.cpu()[:, None]
    if mask is not None:
        keep &= mask.cpu().bool()
    return keep


def check_attention(L, q, k, v, lens=None, mask=None, scale=None, what=()):
    got = L.cross_attention(q, k, v, key_lens=lens, key_mask=mask, scale=scale)
    b, lq, hq, d = q.shape
    lk, hk = k.shape[1], k.shape[2]
    sc = d ** -0.5 if scale is None else scale
    keep = kept_keys(b, lk, lens, mask)
    ref = torch.zeros((b, lq, hq, d), dtype=torch.float64)
    bound = torch.zeros_like(ref)
    u = torch.finfo(q.dtype).eps / 2
    for i in range(b):
        kk, vv = k[i].cpu()[keep[i]].double(), v[i].cpu()[keep[i]].double()
        n = kk.shape[0]
        if n == 0:
            continue
        for h in range(hq):
            j = h // (hq // hk)
            qq = q[i, :, h].double().cpu()
            s = qq @ kk[:, j].t() * sc
            ds = float((qq.abs() @ kk[:, j].abs().t()).max()) * abs(sc) * (d + 4) * 2.0 ** -24
            p = torch.softmax(s, -1)
            ref[i, :, h] = p @ vv[:, j]
            bound[i, :, h] = (np.expm1(2 * ds) + 2 * n * 2.0 ** -24 + 2.0 ** -18 + (u if q.dtype == BF16 else 0)) * 2 * (p @ vv[:, j].abs())
    assert got.dtype == q.dtype and got.is_contiguous()
    within(got, ref, bound * (1 + u) + u * ref.abs() + 1e-38, (q.dtype, tuple(q.shape), tuple(k.shape)) + tuple(what))
    none = ~keep.any(1)
    assert (got.cpu()[none] == 0).all()
    return got


def qkv(t, b, lq, lk, hq, hk, d, seed=40):
    return rand((b, lq, hq, d), t, seed), rand((b, lk, hk, d), t, seed + 1), rand((b, lk, hk, d), t, seed + 2)


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("d", [1, 8, 20, 32, 40, 64, 80, 96, 100, 128, 160, 256])
@pytest.mark.parametrize("lq,lk", [(1, 200), (70, 90)])
def test_attention_head_sizes(L, t, d, lq, lk):
    check_attention(L, *qkv(t, 2, lq, lk, 4, 2, d), what=("d", d))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("b,lq,lk,hq,hk,d", [(1, 1, 1, 1, 1, 64), (1, 1, 3549, 16, 4, 64), (1, 1, 2000, 8, 8, 128), (3, 2, 63, 6, 3, 64), (2, 5, 64, 4, 1, 32),
                                             (2, 33, 65, 2, 2, 64), (1, 127, 300, 3, 1, 64), (2, 129, 129, 2, 1, 128), (1, 300, 1444, 2, 2, 64),
                                             (4, 17, 1, 8, 2, 64), (1, 400, 33, 4, 4, 256), (5, 1, 700, 32, 1, 64), (1, 3, 5776, 2, 1, 128)])
def test_attention_shapes(L, t, b, lq, lk, hq, hk, d):
    check_attention(L, *qkv(t, b, lq, lk, hq, hk, d))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("lq", [1, 3, 40, 200])
@pytest.mark.parametrize("lk", [1, 31, 80, 169, 1000])
def test_attention_masks(L, t, lq, lk):
    b = 6
    q, k, v = qkv(t, b, lq, lk, 4, 2, 64, 50)
    lens = torch.tensor([0, 1, lk, lk + 5, -3, max(1, lk // 2)], dtype=torch.int32).cuda()
    g = torch.Generator().manual_seed(51)
    mask = (torch.rand((b, lk), generator=g) < 0.6)
    mask[1] = False
    mask[2] = True
    mask[3] = False
    mask[3, lk - 1] = True                                        # a single key at the very end
    mask = mask.cuda()
    check_attention(L, q, k, v, lens=lens, what=("lens",))
    check_attention(L, q, k, v, mask=mask, what=("mask",))
    check_attention(L, q, k, v, lens=lens, mask=mask, what=("both",))
    got = L.cross_attention(q, k, v, key_lens=lens.long(), key_mask=mask.to(torch.uint8) * 3)
    assert torch.equal(got, L.cross_attention(q, k, v, key_lens=lens, key_mask=mask))
    # what is left out has no influence, whatever it holds
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(t).min, torch.finfo(t).max):
        k2, v2 = k.clone(), v.clone()
        keep = kept_keys(b, lk, lens, mask).cuda()
        k2[~keep] = bad
        v2[~keep] = bad
        assert torch.equal(L.cross_attention(q, k2, v2, key_lens=lens, key_mask=mask), L.cross_attention(q, k, v, key_lens=lens, key_mask=mask))
        keep = kept_keys(b, lk, lens, None).cuda()
        k2, v2 = k.clone(), v.clone()
        k2[~keep] = bad
        v2[~keep] = bad
        assert torch.equal(L.cross_attention(q, k2, v2, key_lens=lens), L.cross_attention(q, k, v, key_lens=lens))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("d", [136, 160, 192, 248, 256])
@pytest.mark.parametrize("b,lq,lk,hq,hk", [(1, 1, 1, 1, 1), (2, 3, 40, 4, 2), (1, 200, 33, 2, 2), (3, 33, 700, 4, 1), (4, 700, 100, 4, 4)])
def test_attention_wide_heads(L, t, d, b, lq, lk, hq, hk):
    """Head sizes whose values are divided over workgroups, with and without key splits; masked keys hold NaN."""
    q, k, v = qkv(t, b, lq, lk, hq, hk, d, 71)
    check_attention(L, q, k, v, what=(t, d, b, lq, lk))
    keep = torch.rand(b, lk, generator=torch.Generator().manual_seed(4)) < 0.7
    keep[0] = False
    keep = keep.cuda()
    k[~keep] = float("nan")
    v[~keep] = float("nan")
    got = L.cross_attention(q, k, v, key_mask=keep)
    assert torch.isfinite(got).all() and not got[0].any()
    k[~keep] = 0
    v[~keep] = 0
    assert torch.equal(got, L.cross_attention(q, k, v, key_mask=keep))
    check_attention(L, q, k, v, mask=keep, what=("mask", t, d, b, lq, lk))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("lq,lk", [(55, 73), (20, 96), (300, 130)])
def test_attention_several_workgroups_on_a_cu(L, t, d, lq, lk):
    """More workgroups than CUs and more than one tile of keys: neighbours that share a CU do not disturb each other."""
    q, k, v = qkv(t, 30, lq, lk, 16, 4, d, 72)
    lens = torch.randint(lk // 2, lk + 1, (30,), generator=torch.Generator().manual_seed(6), dtype=torch.int32).cuda()
    full = check_attention(L, q, k, v, what=(t, d, lq, lk))
    for _ in range(3):
        assert torch.equal(L.cross_attention(q, k, v), full)
    check_attention(L, q, k, v, lens=lens, what=("lens", t, d, lq, lk))


@pytest.mark.parametrize("t", [BF16, F32])
def test_attention_scales_and_extreme_scores(L, t):
    q, k, v = qkv(t, 2, 50, 333, 4, 4, 64, 60)
    for scale in (0.0, -0.2, 1.0, 3.0):
        check_attention(L, q, k, v, scale=scale, what=("scale", scale))
    # scores that grow along the keys: every tile raises the running maximum; and fall
    for order in (1, -1):
        kk = k.clone()
        kk[:, :, :, 0] = torch.linspace(-40, 40, 333, device="cuda").to(t)[None, :, None] * order
        qq = q.clone()
        qq[..., 0] = 8
        check_attention(L, qq, kk, v, scale=0.25, what=("growing", order))
    # scores around +-1e4 stay finite; a constant score is a mean
    check_attention(L, (q * 0 + 8), (k * 0 + 20), v, scale=1.0, what=("constant",))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("lq,lk,d", [(50, 333, 64), (1, 2000, 32), (300, 700, 128), (7, 90, 5)])
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 15, 2.0 ** 40])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_huge_scores_select_the_largest(L, t, lq, lk, d, size, sign):
    """Scores size^2 * (whole number up to 13) * 0.3, exact before the scale, whose distances are far beyond the range of exp: the
    weights are 1 and 0, so a row is the value of its one largest key (the last, or the second), to one rounding of the quotient."""
    q, k, v = torch.zeros(1, lq, 2, d), torch.zeros(1, lk, 2, d), torch.randn(1, lk, 2, d, generator=torch.Generator().manual_seed(5))
    q[..., 0] = size
    k[..., 0] = size * (torch.arange(lk) % 11).float()[None, :, None]
    k[0, -1, 0, 0], k[0, 1, 1, 0] = 12 * size, 13 * size
    if sign < 0:
        k = -k
    q, k, v = q.to(t).cuda(), k.to(t).cuda(), v.to(t).cuda()
    got = L.cross_attention(q, k, v, scale=0.3 * sign)
    want = torch.stack([v[0, -1, 0], v[0, 1, 1]])[None, None].expand(1, lq, 2, d)
    # exp(0) and the sum are 1 up to the 2^-20 of the exponential's error: the quotient is off by that and the rounding
    bound = want.double().abs() * (2.0 ** -20 + torch.finfo(t).eps / 2)
    within(got, want.double(), bound, (t, lq, lk, d, size, sign))


def test_attention_infinite_scores_follow_the_formula(L):
    """+inf among the kept scores: inf - inf makes the row NaN; -inf: weight zero; all -inf: NaN; other rows untouched."""
    for t in (BF16, F32):
        for lq in (3, 150):
            q, k, v = qkv(t, 1, lq, 200, 2, 2, 64, 70)
            q[0, :, 0, 0] = q[0, :, 0, 0].abs() + 1
            clean = L.cross_attention(q, k, v)
            k2 = k.clone()
            k2[0, 5, 0, 0] = float("inf")
            got = L.cross_attention(q, k2, v)
            assert got[0, :, 0].isnan().all() and torch.equal(got[0, :, 1], clean[0, :, 1])
            k2[0, 5, 0, 0] = -float("inf")
            keep = torch.ones((1, 200), dtype=torch.bool, device="cuda")
            keep[0, 5] = False
            got, without = L.cross_attention(q, k2, v), L.cross_attention(q, k, v, key_mask=keep)
            assert torch.equal(got[0, :, 0], without[0, :, 0])
            k2[0, :, 0, 0] = -float("inf")
            got = L.cross_attention(q, k2, v)
            assert got[0, :, 0].isnan().all() and torch.equal(got[0, :, 1], clean[0, :, 1])


@pytest.mark.parametrize("t", [BF16, F32])
def test_attention_strides_and_alignment(L, t):
    kv = rand((2, 150, 2, 3, 64), t, 80)
    q = rand((2, 6, 40, 64), t, 81).transpose(1, 2)                                # [B, Lq, Hq, D] out of [B, Hq, Lq, D]
    want = check_attention(L, q, kv[:, :, 0], kv[:, :, 1])
    assert torch.equal(want, L.cross_attention(q.contiguous(), kv[:, :, 0].contiguous(), kv[:, :, 1].contiguous()))
    off = rand((2, 150, 3, 69), t, 82)
    check_attention(L, q, off[..., 1:65], kv[:, :, 1])
    check_attention(L, q, kv[:, :, 0], off[..., 2:66])
    check_attention(L, off[:, :40, :, 4:68], kv[:, ::2, 0], kv[:, 1::2, 1])
    one = rand((1, 150, 3, 64), t, 83).expand(2, -1, -1, -1)                       # one image's states for the whole batch
    check_attention(L, q, one, kv[:, :, 1])
    shared = rand((2, 150, 1, 64), t, 84).expand(-1, -1, 3, -1)                    # one head's states for all heads
    check_attention(L, q, shared, shared)
    check_attention(L, rand((64, 40, 3, 2), t, 85).permute(3, 1, 2, 0), kv[:, :, 0], kv[:, :, 1])
    assert L.cross_attention(q[:0], kv[:0, :, 0], kv[:0, :, 1]).shape == (0, 40, 6, 64)
    assert L.cross_attention(q[:, :0], kv[:, :, 0], kv[:, :, 1]).shape == (2, 0, 6, 64)
    assert (L.cross_attention(q, kv[:, :0, 0], kv[:, :0, 1]) == 0).all()


def test_attention_deterministic(L):
    for t in (BF16, F32):
        for lq in (1, 200):
            q, k, v = qkv(t, 3, lq, 1800, 8, 2, 64, 90)
            a = L.cross_attention(q, k, v)
            for _ in range(3):
                assert torch.equal(a, L.cross_attention(q, k, v))


# ---- together, as a head would use them ------------------------------------------------------------------------------------------
def block(L, fm, queries, p, t, key_lens=None):
    """One cross-attention block: object queries over a map's cells (projections, norms + rotation, attention, residuals, MLP)."""
    b, h, w, c = fm.shape
    heads, d = 4, 64
    kv = L.linear(fm, p["kv"], p["kv_b"]).view(b, h * w, 2, heads, d)
    q = L.linear(queries, p["q"]).view(b, -1, heads, d)
    cells = torch.stack(torch.meshgrid(torch.arange(h), torch.arange(w), indexing="ij"), -1).reshape(-1, 2).to(torch.int32).cuda()
    at = torch.arange(q.shape[1], dtype=torch.int32, device="cuda")[:, None].expand(-1, 2)
    qn, kn = L.qk_norm_rope(q, kv[:, :, 0], p["qw"], p["kw"], L.rope_frequencies(d, axes=2), at, cells)
    o = L.cross_attention(qn, kn, kv[:, :, 1], key_lens=key_lens)
    y = L.linear(o.flatten(2), p["o"], residual=queries)
    return L.linear(L.linear(y, p["up"], p["up_b"], activation="gelu"), p["down"], residual=y)


def block_params(c, t):
    e = 256
    r = lambda s, seed, f: rand(s, t, seed, f)  # noqa: E731
    return dict(kv=r((2 * e, c), 100, c ** -0.5), kv_b=r((2 * e,), 101, 0.1), q=r((e, e), 102, e ** -0.5), qw=r((64,), 103, 1), kw=r((64,), 104, 1),
                o=r((e, e), 105, e ** -0.5), up=r((4 * e, e), 106, e ** -0.5), up_b=r((4 * e,), 107, 0.1), down=r((e, 4 * e), 108, (4 * e) ** -0.5))


def block_reference(fm, queries, p, key_lens=None):
    """The same block in float64 without any rounding between the operators."""
    q64 = {k: v.double().cpu() for k, v in p.items()}
    fm, x = fm.double().cpu(), queries.double().cpu()
    b, h, w, c = fm.shape
    kv = (fm.reshape(b, h * w, c) @ q64["kv"].t() + q64["kv_b"]).view(b, h * w, 2, 4, 64)
    q = (x @ q64["q"].t()).view(b, -1, 4, 64)
    f = 10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16).repeat(2)
    cells = torch.stack(torch.meshgrid(torch.arange(h), torch.arange(w), indexing="ij"), -1).reshape(-1, 2)[None]
    at = torch.arange(q.shape[1])[None, :, None].expand(-1, -1, 2)
    qn, _ = ref_norm_rope(q, p["qw"], f, at, 2, False, 1e-6)
    kn, _ = ref_norm_rope(kv[:, :, 0], p["kw"], f, cells, 2, False, 1e-6)
    s = torch.einsum("bqhd,bkhd->bhqk", qn, kn) / 8
    if key_lens is not None:
        s = s.masked_fill(~(torch.arange(h * w)[None, :] < key_lens.cpu()[:, None])[:, None, None], -torch.inf)
    o = torch.einsum("bhqk,bkhd->bqhd", torch.softmax(s, -1), kv[:, :, 1]).flatten(2)
    y = x + o @ q64["o"].t()
    u = y @ q64["up"].t() + q64["up_b"]
    return y + (u * torch.special.ndtr(u)) @ q64["down"].t()


def test_block_over_the_maps_of_the_body(L, oracle, oracle_params):
    """darknet53_body -> the three operators over route_3, float32 and bfloat16, against float64 from the same maps."""
    img = np.random.default_rng(3).random((2, 96, 96, 3), dtype=np.float32)
    with L.variable_scope(oracle_params[:52]):
        fm = L.darknet53_body(img)[2]
    assert fm.shape == (2, 3, 3, 1024)
    fm = fm / fm.std()
    lens = torch.tensor([9, 4], dtype=torch.int32, device="cuda")
    for t, tol in ((F32, 1e-4), (BF16, 6e-2)):
        # tolerance of the chain: float32 in 6 steps of relative error <= 1e-5 each; bf16 rounds ten times (2^-8 each at most) on the longest
        # path, all factors of unit scale: 10 * 2^-8 = 4e-2 of the largest value, and the residual sums carry it once more by half
        p = block_params(1024, t)
        queries = rand((2, 7, 256), t, 110)
        got = block(L, fm.to(t), queries, p, t, lens).double().cpu()
        ref = block_reference(fm.to(t), queries, p, lens)
        assert float((got - ref).abs().max()) <= tol * float(ref.abs().max())
        # one query at a time over the same states: a step gives the row of the whole call
        if t == F32:
            one = block(L, fm, queries[:, :1], p, t, lens).double().cpu()
            assert float((one - ref[:, :1]).abs().max()) <= tol * float(ref.abs().max())


def test_streams_and_graphs(L):
    """A block captured once and replayed on new inputs, with eager calls between the replays, and two captures side by side."""
    t = BF16
    p = block_params(256, t)
    fms = [rand((2, 13, 13, 256), t, 120 + i) for i in range(6)]
    qs = [rand((2, 5, 256), t, 130 + i) for i in range(6)]
    cells = torch.stack(torch.meshgrid(torch.arange(13), torch.arange(13), indexing="ij"), -1).reshape(-1, 2).to(torch.int32).cuda()
    at, f = torch.arange(5, dtype=torch.int32, device="cuda"), L.rope_frequencies(64, axes=2)
    at2 = at[:, None].expand(-1, 2).contiguous()

    def step(fm, queries):
        kv = L.linear(fm, p["kv"], p["kv_b"]).view(2, 169, 2, 4, 64)
        qn, kn = L.qk_norm_rope(L.linear(queries, p["q"]).view(2, 5, 4, 64), kv[:, :, 0], p["qw"], p["kw"], f, at2, cells)
        return L.linear(L.cross_attention(qn, kn, kv[:, :, 1]).flatten(2), p["o"], residual=queries)

    want = [step(a, b) for a, b in zip(fms, qs)]
    graphs = []
    for i in range(2):
        bufs = (fms[0].clone(), qs[0].clone())
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            out = step(*bufs)
        graphs.append((g, bufs, out))
    for i in range(6):
        for n, (g, (bf, bq), out) in enumerate(graphs):
            j = (i + 3 * n) % 6
            bf.copy_(fms[j])
            bq.copy_(qs[j])
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        graphs[0][0].replay()
        eager = step(fms[i], qs[i])
        torch.cuda.synchronize()
        assert torch.equal(eager, want[i])
        for n, (g, _, out) in enumerate(graphs):
            assert torch.equal(out, want[(i + 3 * n) % 6]), (i, n)


def test_refusals(L):
    x, w = rand((3, 8), BF16, 140), rand((4, 8), BF16, 141)
    bad = [lambda: L.linear(x, w.float()), lambda: L.linear(x, w[:, :7]), lambda: L.linear(x.half(), w.half()), lambda: L.linear(x, w, activation="tanh"),
           lambda: L.linear(x, w, x[0]), lambda: L.linear(x, w, residual=x), lambda: L.linear(x, w, residual=rand((3, 4), F32, 1)),
           lambda: L.linear(x, w[:0]), lambda: L.linear(x, w.clone().requires_grad_()), lambda: L.linear(x[:, :0], w[:, :0])]
    q, k, v = qkv(BF16, 2, 3, 5, 4, 2, 64)
    bad += [lambda: L.cross_attention(q, k, v[:, :4]), lambda: L.cross_attention(q, k.float(), v), lambda: L.cross_attention(q[:, :, :3], k, v),
            lambda: L.cross_attention(q[:1], k, v), lambda: L.cross_attention(q, k, v, key_lens=torch.ones(3, dtype=torch.int32)),
            lambda: L.cross_attention(q, k, v, key_lens=torch.ones(2)), lambda: L.cross_attention(q, k, v, key_mask=torch.ones(2, 4, dtype=torch.bool)),
            lambda: L.cross_attention(q, k, v, key_mask=torch.ones(2, 5)), lambda: L.cross_attention(q[0], k, v),
            lambda: L.cross_attention(rand((1, 1, 1, 264), F32, 1), rand((1, 1, 1, 264), F32, 1), rand((1, 1, 1, 264), F32, 1)),
            lambda: L.cross_attention(q.clone().requires_grad_(), k, v)]
    f, p = L.rope_frequencies(64), torch.arange(3)
    bad += [lambda: L.qk_norm_rope(q, k, frequencies=f, q_positions=p), lambda: L.qk_norm_rope(q, None, frequencies=f),
            lambda: L.qk_norm_rope(q, None, frequencies=f, q_positions=p.float()), lambda: L.qk_norm_rope(q, None, frequencies=f, q_positions=p[:2]),
            lambda: L.qk_norm_rope(q, None, frequencies=L.rope_frequencies(66), q_positions=p), lambda: L.qk_norm_rope(q, None, q_weight=f[:3]),
            lambda: L.qk_norm_rope(q, None, eps=0.0), lambda: L.qk_norm_rope(q, k[:1]), lambda: L.qk_norm_rope(q, k.float()),
            lambda: L.qk_norm_rope(q, k, rand((64,), BF16, 1), rand((64,), F32, 1)), lambda: L.rope_frequencies(7), lambda: L.rope_frequencies(6, axes=2),
            lambda: L.qk_norm_rope(q[:, :2], None, frequencies=f, q_positions=torch.zeros((2, 2), dtype=torch.int32)),
            lambda: L.qk_norm_rope(q, None, frequencies=f[:31], q_positions=torch.zeros((3, 2), dtype=torch.int32), axes=2)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail("call %d was accepted" % i)
    with torch.no_grad():
        assert torch.equal(L.linear(x, w.clone().requires_grad_()), L.linear(x, w))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("b,lq,lk,hq,hk,d", [(1, 1, 40000, 4, 4, 64), (1, 2, 33333, 8, 2, 128), (2, 40, 20001, 2, 1, 64), (1, 1, 9000, 2, 2, 256), (3, 1, 15000, 2, 1, 32)])
def test_attention_long_states(L, t, b, lq, lk, hq, hk, d):
    """Few queries over long states: the keys are split over workgroups and joined."""
    q, k, v = qkv(t, b, lq, lk, hq, hk, d, 95)
    check_attention(L, q, k, v)
    lens = torch.tensor([lk - 7, 0, lk // 3][:b], dtype=torch.int32, device="cuda")
    check_attention(L, q, k, v, lens=lens, what=("lens",))
    k[:, lk // 2:, 0, 0] = float("nan")
    keep = torch.ones((b, lk), dtype=torch.bool, device="cuda")
    keep[:, lk // 2:] = False
    keep[:, 3] = False
    v[:, 3] = float("inf")
    check_attention(L, q, k, v, lens=lens, mask=keep, what=("both",))
    k[:, 5, 0, 0] = float("nan")
    got = L.cross_attention(q, k, v, key_mask=keep)
    assert got[:, :, :hq // hk].isnan().all()
    if hk > 1:
        assert torch.isfinite(got[:, :, hq // hk:]).all()


def test_split_attention_in_graphs_on_two_streams(L):
    """Key splits use a workspace: two captured graphs and eager calls on other streams at the same time keep to their own."""
    cases = [qkv(BF16, 2, 1, 6000, 8, 2, 64, 200), qkv(F32, 1, 90, 4000, 4, 4, 64, 210)]
    from yolo_amd import _lib
    for code, (q, k, v) in zip((1, 0), cases):
        assert _lib.lib().yolo_cross_attention_workspace_bytes(code, q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], 64) > 0
    want = [L.cross_attention(*c) for c in cases]
    graphs = []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = L.cross_attention(*c)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, out in graphs:
            out.zero_()
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = [L.cross_attention(*c) for c in cases]
        here = [L.cross_attention(*c) for c in cases]
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(graphs[i][1], want[i]) and torch.equal(eager[i], want[i]) and torch.equal(here[i], want[i])


def test_attention_workspace_is_checked(L):
    """The C entry: too small a workspace is an error before any launch; an unaligned call needs none."""
    import ctypes
    from yolo_amd import _lib, _tensor
    lib = _lib.lib()
    q, k, v = qkv(BF16, 1, 1, 6000, 2, 2, 64, 220)
    need = lib.yolo_cross_attention_workspace_bytes(1, 1, 1, 6000, 2, 2, 64)
    st = (ctypes.c_int64 * 3)(k.stride(0), k.stride(1), k.stride(2))
    qs = (ctypes.c_int64 * 3)(q.stride(0), q.stride(1), q.stride(2))
    out, ws = torch.zeros_like(q), _tensor.workspace(need)

    def call(w, n):
        return lib.yolo_cross_attention(1, q.data_ptr(), qs, k.data_ptr(), st, v.data_ptr(), st, None, None, 1, 1, 6000, 2, 2, 64, 0.125,
                                        out.data_ptr(), w, n, _tensor.stream_ptr())
    assert call(None, 0) == -5 and call(ws.data_ptr(), need - 1) == -5 and call(ws.data_ptr() + 8, need) == -5
    assert b"workspace" in lib.yolo_last_error() and (out == 0).all()
    assert call(ws.data_ptr(), need) == 0
    assert torch.equal(out, L.cross_attention(q, k, v))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("d,r", [(64, 16), (64, 32), (64, 48), (96, 64), (128, 32), (256, 128), (80, 16), (48, 40)])
def test_qk_partial_rotation(L, t, d, r):
    """rotary_dim below the head size, in whole pieces (register kernel) and not (general one)."""
    q, k = rand((2, 21, 5, d), t, 230), rand((2, 33, 2, d), t, 231)
    f, w = L.rope_frequencies(r, axes=2), rand((d,), t, 232)
    for il in (False, True):
        check_qk(L, q, k, w, w, f, grid_positions(21, 2, 2, 3), grid_positions(33, 2, 2), 2, il)


def test_unaligned_attention_through_the_c_entry(L):
    """Rows off 16-byte boundaries straight into the C entry (the Python function copies them): the general kernel, no workspace."""
    import ctypes
    from yolo_amd import _lib, _tensor
    for t, code in ((F32, 0), (BF16, 1)):
        big = rand((2, 70, 3, 67), t, 240)
        q, k, v = big[:, :9, :, 1:65], big[:, 9:, :, 2:66], big[:, 9:, :, 3:67]
        st = [(ctypes.c_int64 * 3)(*x.stride()[:3]) for x in (q, k, v)]
        lens, mask = torch.tensor([61, 20], dtype=torch.int32, device="cuda"), torch.ones((2, 61), dtype=torch.bool, device="cuda")
        mask[0, ::3] = False
        out = torch.full((2, 9, 3, 64), 9.0, dtype=t, device="cuda")
        _lib.check(_lib.lib().yolo_cross_attention(code, q.data_ptr(), st[0], k.data_ptr(), st[1], v.data_ptr(), st[2], lens.data_ptr(),
                                                   mask.data_ptr(), 2, 9, 61, 3, 3, 64, 0.125, out.data_ptr(), None, 0, _tensor.stream_ptr()))
        want = L.cross_attention(q, k, v, key_lens=lens, key_mask=mask)
        # the two kernels differ by their roundings: one of the result and, in bf16, one of each weight
        u = torch.finfo(t).eps / 2
        a = L.cross_attention(q, k, v.abs(), key_lens=lens, key_mask=mask).double()
        within(out, want.double(), 2 * u * want.double().abs() + (2.0 ** -16 + (2 * u if t == BF16 else 0)) * 2 * a, t)


def test_offsets_past_32_bits(L):
    """Strides and sizes whose byte offsets pass 2^32: a state cache with far rows, wide rows of a matrix product, a result of more than
    2^32 bytes."""
    buf = torch.zeros(3_000_000_000, dtype=BF16, device="cuda")                    # 6 GB
    far = buf.as_strided((1, 700, 2, 64), (0, 4_000_000, 64, 1))
    q, k, v = qkv(BF16, 1, 5, 700, 4, 2, 64, 250)
    far.copy_(k)
    want = L.cross_attention(q, k, v)
    assert torch.equal(L.cross_attention(q, far, v), want)
    for lq in (1, 300):                                                            # one-wave and four-wave tiles
        ql = rand((1, lq, 4, 64), BF16, 251)
        assert torch.equal(L.cross_attention(ql, far, far), L.cross_attention(ql, k, k))
    f, p = L.rope_frequencies(64), torch.arange(700, device="cuda")
    assert torch.equal(L.qk_norm_rope(far, None, None, None, f, p)[0], L.qk_norm_rope(k, None, None, None, f, p)[0])
    assert torch.equal(L.qk_norm_rope(far[..., :40], None)[0], L.qk_norm_rope(k[..., :40], None)[0])    # general kernel
    x = far[0, :, 0]                                                               # rows 8 MB apart
    w = rand((1000, 64), BF16, 252)
    assert torch.equal(L.linear(x, w), L.linear(k[0, :, 0], w)) or torch.allclose(L.linear(x, w).float(), L.linear(k[0, :, 0], w).float(), rtol=2 ** -7, atol=2 ** -16)
    del buf, far, x
    x, w = rand((70_000, 16), BF16, 253), rand((32_768, 16), BF16, 254)
    y = L.linear(x, w)                                                             # 4.6 GB
    for rows in (slice(0, 64), slice(65_500, 65_600), slice(69_950, 70_000)):
        check = x[rows].double().cpu() @ w.double().cpu().t()
        assert ((y[rows].double().cpu() - check).abs() <= 2.0 ** -8 * check.abs() + 2.0 ** -18 * 64).all()


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("d", [1, 7, 20, 63, 100, 255])
def test_attention_odd_head_sizes_through_the_c_entry(L, t, d):
    """Any head size straight into the C entry (the Python function pads it): the general kernel, with lens and a mask."""
    import ctypes
    from yolo_amd import _lib, _tensor
    q, k, v = qkv(t, 2, 5, 130, 4, 2, d, 260)
    lens = torch.tensor([130, 67], dtype=torch.int32, device="cuda")
    mask = torch.ones((2, 130), dtype=torch.bool, device="cuda")
    mask[1, ::5] = False
    st = [(ctypes.c_int64 * 3)(*x.stride()[:3]) for x in (q, k, v)]
    assert _lib.lib().yolo_cross_attention_workspace_bytes(0, 2, 5, 130, 4, 2, d) == 0

    def call(q, k, v, key_lens, key_mask, scale):
        out = torch.full((2, 5, 4, d), 9.0, dtype=t, device="cuda")
        _lib.check(_lib.lib().yolo_cross_attention(0 if t == F32 else 1, q.data_ptr(), st[0], k.data_ptr(), st[1], v.data_ptr(), st[2],
                                                   key_lens.data_ptr(), key_mask.data_ptr(), 2, 5, 130, 4, 2, d, d ** -0.5, out.data_ptr(), None, 0,
                                                   _tensor.stream_ptr()))
        return out

    class Entry:
        cross_attention = staticmethod(call)
    check_attention(Entry, q, k, v, lens, mask, what=("c entry", d))
    check_attention(L, q, k, v, lens, mask, what=("padded", d))


@pytest.mark.parametrize("t", [BF16, F32])
@pytest.mark.parametrize("n", [16, 640])                       # the direct kernel and a tile kernel
def test_gelu_is_relatively_exact_in_the_negative_tail(L, t, n):
    """Every bfloat16 from -2^-10 to -12.75 as an exact pre-activation: the result is within its rounding and 2^-13 of y itself (bfloat16: the
    formula is within 2^-14; float32: the error function's sixteen last places at most), and v^2 2^-22 of y for the rounded argument
    of the exponential: v^2 / 2 times four roundings of 2^-24."""
    v = -(torch.arange(int(12.75 * 2 ** 7), 0, -1).double() * 2.0 ** -7)            # to -2^-7 ..
    v = torch.cat([v, -(torch.arange(128, 256).double()[:, None] * 2.0 ** -torch.arange(7, 18).double()).flatten()]).to(BF16).to(t).cuda()      # .. octaves to -2^-10
    x, w = torch.zeros((v.numel(), 8), dtype=t, device="cuda"), torch.zeros((n, 8), dtype=t, device="cuda")
    x[:, 0], w[:, 0] = v, 1
    v64 = v.double().cpu()
    y = v64 * 0.5 * torch.special.erfc(-v64 * 0.5 ** 0.5)      # torch's ndtr is 1 + erf, which leaves nothing of the tail below -8.3
    u, formula = torch.finfo(t).eps / 2, 2.0 ** -13 if t == BF16 else 2.0 ** -19
    bound = (u * (1 + formula) + formula + v64 * v64 * 2.0 ** -22) * y.abs() + 1e-38
    got = L.linear(x, w, activation="gelu")
    within(got, y[:, None].expand(-1, n), bound[:, None].expand(-1, n), (t, n))


@pytest.mark.parametrize("b,lq,lk,hq,hk,d", [(1, 1, 3549, 16, 4, 64), (2, 3, 200, 8, 2, 128), (3, 8, 300, 4, 1, 32), (1, 32, 150, 2, 2, 96), (1, 5, 400, 2, 1, 256),
                                             (300, 1, 200, 16, 4, 64), (600, 2, 130, 4, 2, 32), (1, 1, 900, 4, 4, 200)])
def test_attention_of_few_queries_keeps_whole_weights(L, b, lq, lk, hq, hk, d):
    """bfloat16 with up to 32 rows a head group: the weights are the upper 16 bits and the rest rounded to bfloat16.  Cutting leaves less than 2^-7
    of a weight, and rounding that is off by 2^-8 of it: 2^-15 of a weight where one rounding to bfloat16 is 2^-8."""
    q, k, v = qkv(BF16, b, lq, lk, hq, hk, d, 300)
    got = L.cross_attention(q, k, v)
    g, u = hq // hk, torch.finfo(BF16).eps / 2
    q64, k64, v64 = (x.double().cpu() for x in (q, k, v))
    for i in range(0, b, max(1, b // 20)):
        for h in range(hq):
            qq, kk, vv = q64[i, :, h], k64[i, :, h // g], v64[i, :, h // g]
            ds = float((qq.abs() @ kk.abs().t()).max()) * d ** -0.5 * (d + 4) * 2.0 ** -24
            p = torch.softmax(qq @ kk.t() * d ** -0.5, -1)
            ref = p @ vv
            bound = (np.expm1(2 * ds) + 2 * lk * 2.0 ** -24 + 2.0 ** -18 + 2.0 ** -15) * 2 * (p @ vv.abs())
            within(got[i, :, h], ref, bound * (1 + u) + u * ref.abs(), (b, lq, lk, hq, hk, d, i, h))
