"""Block-scaled 8-bit products, rotary positions and group normalisation against 64-bit forms (needs a B200).

Tolerances count roundings: an output is off by at most half a step of its type, eps/2 relative to the
value (plus half of the smallest subnormal), and by what the fp32 arithmetic before it may be off, a
number of 2^-24 steps of the magnitudes that were added.
"""

import math

import pytest
import torch

from zimage_b200 import (Fp8BlockLinear, GroupNormAct, _lib, fp8_block_linear, fp8_block_matmul, fp8_block_quantize,
                         fp8_block_quantize_weight, fp8_block_transpose, group_norm_act, rotary_embed, rotary_table)

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def check(got, ref, extra):
    """|got - ref| <= half a step of got's type at ref, plus `extra` (fp32 error before that rounding)."""
    info = torch.finfo(got.dtype)
    lim = (ref.abs() + extra) * (info.eps / 2) + extra + info.smallest_normal * info.eps / 2
    bad = (got.double() - ref).abs() > lim
    # from half a step over the largest value on (65520 in fp16), rounding gives an infinity of that sign
    over = torch.isinf(got) & (ref.abs() + extra >= info.max * (1 + info.eps / 4)) & (got.sign() == ref.sign())
    bad &= ~over
    bad |= torch.isnan(got) != torch.isnan(ref)
    assert got.shape == ref.shape
    assert not bad.any(), (int(bad.sum()), float((got.double() - ref).abs().max()))


# --- 8-bit quantisation -------------------------------------------------------------------------


def ref_scale(amax):
    """The least 2^e, e >= -120, with amax <= 448 * 2^e, by its definition."""
    e = torch.full_like(amax, -120.0)
    for _ in range(260):
        e = torch.where(amax > 448.0 * torch.exp2(e), e + 1, e)
    return torch.exp2(e)


def ref_e4m3(v):
    """Nearest value of the e4m3 grid, ties to even: 3 bits after the leading one, none finer than 2^-9."""
    _, ex = torch.frexp(v.abs().clamp(min=2.0 ** -20))  # v = m 2^ex, m in [1/2, 1)
    step = torch.exp2((ex.double() - 4).clamp(min=-9.0))
    return torch.round(v / step) * step


def ref_rows(x):
    M, K = x.shape
    kb = -(-K // 128)
    xd = torch.nn.functional.pad(x.double(), (0, kb * 128 - K)).view(M, kb, 128)
    bad = ~torch.isfinite(xd).all(-1)
    xd = torch.where(bad[..., None], torch.ones_like(xd), xd)
    s = ref_scale(xd.abs().amax(-1))
    q = ref_e4m3(xd / s[..., None])
    q[bad], s[bad] = math.nan, math.nan
    return q.view(M, kb * 128)[:, :K], s


def ref_blocks(w):
    N, K = w.shape
    nb, kb = -(-N // 128), -(-K // 128)
    wd = torch.nn.functional.pad(w.double(), (0, kb * 128 - K, 0, nb * 128 - N)).view(nb, 128, kb, 128)
    s = ref_scale(wd.abs().amax((1, 3)))
    q = ref_e4m3(wd / s[:, None, :, None])
    return q.view(nb * 128, kb * 128)[:N, :K], s


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=12345.0), torch.nan_to_num(b.double(), nan=12345.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 129), (77, 640), (130, 3840), (5, 1000), (64, 72), (9, 10240)])
def test_quantise_rows_exact(cuda, dtype, M, K):
    g = _gen(M + K)
    x = _randn(g, M, K) * torch.exp2(torch.randint(-12, 12, (M, K), generator=g, device="cuda").float())
    x = x.to(dtype)
    x[0, : K // 2] = 0
    if M > 4:
        x[1] = 448.0  # exactly the largest value
        x[2] = 449.0 if dtype != torch.bfloat16 else 452.0
        x[3] = torch.finfo(dtype).max
        x[4] = torch.finfo(dtype).smallest_normal / 4
    q, s = fp8_block_quantize(x)
    rq, rs = ref_rows(x)
    assert q.dtype == torch.float8_e4m3fn and same(q, rq) and same(s, rs)


def test_quantise_ties_and_every_e4m3_midpoint(cuda):
    """Midpoints between neighbouring e4m3 values round to the even one; every bf16 in reach is right."""
    bits = torch.arange(0x7F80, dtype=torch.int32, device="cuda").to(torch.int16)
    x = bits.view(torch.bfloat16)
    x = x[x <= 448.0]
    pad = (-x.numel()) % 127
    x = torch.cat([x, x.new_zeros(pad)]).view(-1, 127)
    x = torch.cat([x, x.new_full((x.shape[0], 1), 448.0)], 1)  # scale 1 in every row
    x = torch.cat([x, -x])
    q, s = fp8_block_quantize(x)
    assert bool((s == 1).all())
    assert same(q, ref_e4m3(x.double()))


def test_quantise_non_finite_blocks(cuda):
    x = _randn(_gen(3), 4, 384).to(torch.bfloat16)
    x[0, 5], x[1, 200], x[2, 383] = math.inf, math.nan, -math.inf
    q, s = fp8_block_quantize(x)
    rq, rs = ref_rows(x)
    assert same(q, rq) and same(s, rs)
    assert int(torch.isnan(s).sum()) == 3


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (200, 333), (257, 1000), (640, 384)])
def test_quantise_weight_exact(cuda, dtype, N, K):
    w = (_randn(_gen(N), N, K) * torch.exp2(torch.arange(K, device="cuda") % 9 - 4.0)).to(dtype)
    q, s = fp8_block_quantize_weight(w)
    rq, rs = ref_blocks(w)
    assert same(q, rq) and same(s, rs)
    t = fp8_block_transpose(q)
    assert same(t, rq.t())


def test_quantise_leading_dimensions_and_strides(cuda):
    x = _randn(_gen(1), 3, 5, 320).to(torch.bfloat16)
    q, s = fp8_block_quantize(x)
    q2, s2 = fp8_block_quantize(x.view(15, 320))
    assert q.shape == (3, 5, 320) and s.shape == (3, 5, 3)
    assert same(q.reshape(15, 320), q2) and same(s.reshape(15, 3), s2)
    v = fp8_block_quantize(x[0, 0])
    assert v[0].shape == (320,) and v[1].shape == (3,) and same(v[0], q2[0])
    sliced = x[:, 1:4, 7:200]  # odd offset, strided rows
    qs, ss = fp8_block_quantize(sliced)
    rq, rs = ref_rows(sliced.reshape(9, 193))
    assert same(qs.reshape(9, 193), rq) and same(ss.reshape(9, 2), rs)
    e = fp8_block_quantize(x[:0])
    assert e[0].shape == (0, 5, 320) and e[1].shape == (0, 5, 3)


# --- the product --------------------------------------------------------------------------------


def product_terms(qx, sx, qw, sw):
    """(exact product, sum of magnitudes) of dequantised operands."""
    K, N = qx.shape[1], qw.shape[0]
    a = qx.double() * sx.double().repeat_interleave(128, 1)[:, :K]
    b = qw.double() * sw.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return a @ b.t(), a.abs() @ b.abs().t()


def product_extra(mag, K, bias=None):
    # at most K - 1 additions and the scale products, each within one step of the sum of magnitudes
    e = (K + 8) * U32 * mag
    return e if bias is None else e + U32 * (mag + bias.double().abs())


SHAPES = [(1, 128, 128), (1, 3840, 500), (2, 640, 136), (7, 1000, 257), (8, 256, 1024), (9, 512, 384), (16, 3840, 136),
          (33, 384, 128), (64, 130, 64), (127, 256, 129), (128, 128, 256), (129, 768, 300), (300, 2560, 640),
          (513, 1024, 1300), (1, 17, 3), (260, 16, 8), (1030, 640, 1920), (2, 10240, 64), (700, 4992, 328)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_forward(cuda, dtype, M, K, N):
    g = _gen(M * 7 + K + N)
    x = _randn(g, M, K).to(dtype)
    x[:, :: 61] *= 20
    wq, ws = fp8_block_quantize_weight(_randn(g, N, K).to(torch.bfloat16) * 0.05)
    bias = _randn(g, N).to(dtype) if N % 2 else None
    y = fp8_block_linear(x, wq, ws, bias)
    ref, mag = product_terms(*ref_rows(x), wq, ws)
    check(y, ref if bias is None else ref + bias.double(), product_extra(mag, K, bias))
    assert _lib.device_error_read_clear() == 0


@pytest.mark.parametrize("M,K,N", [(1, 384, 200), (5, 700, 130), (40, 512, 256), (200, 1100, 520), (600, 640, 384)])
def test_matmul_any_scales(cuda, M, K, N):
    """Scales that are no powers of two, of any sign, strided and broadcast."""
    g = _gen(K)
    xq, _ = fp8_block_quantize(_randn(g, M, K))
    wq, _ = fp8_block_quantize_weight(_randn(g, N, K))
    nb, kb = -(-N // 128), -(-K // 128)
    sx = _randn(g, kb, M).t() * 0.3
    sw = _randn(g, nb, 2 * kb)[:, ::2] * 0.7
    y = fp8_block_matmul(xq, sx, wq, sw, out_dtype=torch.float32)
    ref, mag = product_terms(xq, sx, wq, sw)
    check(y, ref, product_extra(mag, K))
    one = torch.full((1, 1), 0.37, device="cuda").expand(M, kb)
    y = fp8_block_matmul(xq.contiguous()[:, :K], one, wq, sw, out_dtype=torch.float16)
    ref, mag = product_terms(xq, one, wq, sw)
    check(y, ref, product_extra(mag, K))


@pytest.mark.parametrize("M", [1, 6, 70, 400])
def test_product_sums_are_kept_in_32_bits(cuda, M):
    """A large term that cancels leaves the small ones: within a block and across blocks."""
    K, N = 1024, 256
    x = torch.full((M, K), 2.0 ** -6, device="cuda")
    x[:, 0], x[:, 1] = 448.0, -448.0         # same block
    x[:, 256], x[:, 384] = 256.0, -256.0     # different blocks
    xq = x.to(torch.float8_e4m3fn)
    wq = torch.ones(N, K, device="cuda").to(torch.float8_e4m3fn)
    sx = torch.ones(M, K // 128, device="cuda")
    sw = torch.ones(N // 128, K // 128, device="cuda")
    y = fp8_block_matmul(xq, sx, wq, sw, out_dtype=torch.float32)
    want = (K - 4) * 2.0 ** -6
    # products are multiples of 2^-6 below 2^9: 15 bits, so every partial sum is exact in 32 bits
    assert bool((y == want).all()), float((y - want).abs().max())


@pytest.mark.parametrize("M", [1, 8, 9, 16, 17, 300])
def test_linear_sums_are_kept_in_32_bits(cuda, M):
    """The same through the linear, whose few-token form sums on other instructions: values that the
    quantiser holds exactly (448 gives a block the scale 1)."""
    K, N = 1024, 256
    x = torch.full((M, K), 2.0 ** -6, device="cuda")
    x[:, ::128], x[:, 1::128] = 448.0, -448.0
    x[:, 3], x[:, 260] = 256.0, -256.0
    y = fp8_block_linear(x, torch.ones(N, K, device="cuda").to(torch.float8_e4m3fn), torch.ones(2, 8, device="cuda"))
    assert bool((y == (K - 18) * 2.0 ** -6).all()), float((y - (K - 18) * 2.0 ** -6).abs().max())


@pytest.mark.parametrize("M", [1, 5, 40])
def test_linear_of_one_row_dimensions(cuda, M):
    """Views whose dimensions of one element carry strides of their own."""
    g = _gen(3)
    wq, ws = fp8_block_quantize_weight(_randn(g, 130, 256))
    x = _randn(g, 1, M, 256).to(torch.bfloat16)
    want = fp8_block_linear(x[0], wq, ws)
    assert torch.equal(fp8_block_linear(x.transpose(0, 1), wq, ws)[:, 0], want)
    xs = x.transpose(0, 1).detach().requires_grad_()
    d = _randn(g, 1, M, 130).to(torch.bfloat16)
    (dx,) = torch.autograd.grad(fp8_block_linear(xs, wq, ws), (xs,), d.transpose(0, 1))
    x0 = x[0].detach().requires_grad_()
    (d0,) = torch.autograd.grad(fp8_block_linear(x0, wq, ws), (x0,), d[0])
    assert torch.equal(dx[:, 0], d0)
    wide = _randn(g, M, 300).to(torch.bfloat16)[:, 8:264]
    assert torch.equal(fp8_block_linear(wide, wq, ws), fp8_block_linear(wide.contiguous(), wq, ws))


@pytest.mark.parametrize("M,at", [(4, (2, 300)), (150, (149, 0)), (600, (300, 639))])
def test_linear_non_finite_rows_stay_apart(cuda, M, at):
    K, N = 640, 256
    x = _randn(_gen(M), M, K).to(torch.bfloat16)
    x[at] = math.inf
    wq, ws = fp8_block_quantize_weight(_randn(_gen(1), N, K))
    y = fp8_block_linear(x, wq, ws)
    bad = torch.isnan(y)
    assert bool(bad[at[0]].all()) and int(bad.sum()) == N


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 256, 128), (5, 640, 300), (130, 384, 640), (333, 1000, 520), (64, 130, 257)])
@pytest.mark.parametrize("laid_out", [False, True])
def test_linear_gradients(cuda, dtype, M, K, N, laid_out):
    g = _gen(M + K + N)
    x = _randn(g, M, K).to(dtype).requires_grad_()
    wq, ws = fp8_block_quantize_weight(_randn(g, N, K).to(torch.bfloat16) * 0.05)
    bias = _randn(g, N).to(dtype).requires_grad_()
    dy = _randn(g, M, N).to(dtype)
    y = fp8_block_linear(x, wq, ws, bias, w_q_t=fp8_block_transpose(wq) if laid_out else None)
    dx, db = torch.autograd.grad(y, (x, bias), dy)
    ref, mag = product_terms(*ref_rows(dy), wq.t(), ws.t())
    check(dx, ref, product_extra(mag, N))
    check(db, dy.double().sum(0), (M + 2) * U32 * dy.double().abs().sum(0))
    # one of the two alone, and a gradient that is an expanded view
    y = fp8_block_linear(x.detach(), wq, ws, bias)
    (db1,) = torch.autograd.grad(y.sum(), (bias,))
    assert torch.equal(db1, torch.full_like(db1, float(M)))
    (dx1,) = torch.autograd.grad(fp8_block_linear(x, wq, ws).sum(), (x,))
    ref, mag = product_terms(*ref_rows(torch.ones_like(dy)), wq.t(), ws.t())
    check(dx1, ref, product_extra(mag, N))


def test_linear_gradient_against_differences(cuda):
    """With values the format holds exactly the forward map is linear, so differences give its slope."""
    K, N, M = 256, 96, 3
    g = _gen(5)
    x = torch.randint(-8, 9, (M, K), generator=g, device="cuda").float()
    x[:, ::128] = 256.0  # keeps every block's scale at 1 while another value moves
    wq, ws = fp8_block_quantize_weight(torch.randint(-4, 5, (N, K), generator=g, device="cuda").float())
    dy = torch.randint(-4, 5, (M, N), generator=g, device="cuda").float()
    x.requires_grad_()
    (dx,) = torch.autograd.grad(fp8_block_linear(x, wq, ws), (x,), dy)
    for m, k in ((0, 1), (1, 130), (2, 255)):
        up, dn = x.detach().clone(), x.detach().clone()
        up[m, k] += 1
        dn[m, k] -= 1
        diff = ((fp8_block_linear(up, wq, ws) - fp8_block_linear(dn, wq, ws)) * dy).double().sum() / 2
        assert float(diff) == float(dx[m, k])


def test_linear_empty_and_leading_dimensions(cuda):
    wq, ws = fp8_block_quantize_weight(_randn(_gen(1), 200, 256))
    assert fp8_block_linear(torch.empty(0, 256, device="cuda"), wq, ws).shape == (0, 200)
    x = torch.empty(2, 0, 256, device="cuda", requires_grad=True)
    b = torch.zeros(200, device="cuda", requires_grad=True)
    y = fp8_block_linear(x, wq, ws, b)
    dx, db = torch.autograd.grad(y.sum(), (x, b))
    assert y.shape == (2, 0, 200) and dx.shape == x.shape and bool((db == 0).all())
    x = _randn(_gen(2), 2, 3, 256)
    y = fp8_block_linear(x, wq, ws)
    assert torch.equal(y.view(6, 200), fp8_block_linear(x.view(6, 256), wq, ws))
    assert torch.equal(y[0, 0], fp8_block_linear(x[0, 0], wq, ws))
    assert torch.equal(fp8_block_linear(x.transpose(0, 1), wq, ws), y.transpose(0, 1))


def test_linear_weight_views(cuda):
    """A weight with odd strides and an odd offset gives what its copy gives, call after call."""
    g = _gen(9)
    big = _randn(g, 300, 700).to(torch.float8_e4m3fn)
    w = big[7:263, 3:643]
    ws = torch.rand(2, 5, generator=g, device="cuda")
    x = _randn(g, 40, 640).to(torch.bfloat16)
    y = fp8_block_linear(x, w, ws)
    assert torch.equal(y, fp8_block_linear(x, w.contiguous(), ws))
    assert torch.equal(y, fp8_block_linear(x, w, ws))


# --- rotary positions ---------------------------------------------------------------------------


def ref_rotary(x, cos, sin, layout):
    """x [B, S, H, D], cos/sin [B, S, R/2] in fp64; also the magnitudes added."""
    half = cos.shape[-1]
    v = x.double().clone()
    c, s = cos.double()[:, :, None], sin.double()[:, :, None]
    ia = slice(0, half) if layout == "half" else slice(0, 2 * half, 2)
    ib = slice(half, 2 * half) if layout == "half" else slice(1, 2 * half, 2)
    a, b = v[..., ia].clone(), v[..., ib].clone()
    mag = torch.zeros_like(v)
    v[..., ia], v[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia], mag[..., ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return v, mag


def table(L, half, seed=0):
    ang = torch.rand(L, half, generator=_gen(seed), device="cuda") * 20 - 10
    return ang.cos(), ang.sin()


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,H,Hk,D,R", [(1, 1, 1, 0, 2, 2), (2, 3, 5, 2, 128, 128), (1, 17, 3, 3, 128, 64),
                                          (3, 4, 2, 1, 80, 80), (1, 9, 4, 2, 48, 24), (2, 5, 3, 1, 34, 10),
                                          (1, 300, 30, 30, 128, 128), (1, 6, 2, 2, 1024, 1024), (2, 7, 6, 2, 256, 192)])
def test_rotary_forward_and_gradient(cuda, layout, dtype, B, S, H, Hk, D, R):
    g = _gen(D + S)
    q = _randn(g, B, S, H, D).to(dtype).requires_grad_()
    k = _randn(g, B, S, Hk, D).to(dtype).requires_grad_() if Hk else None
    cos, sin = table(S + 11, R // 2)
    pos = torch.randint(0, S + 11, (B, S), generator=g, device="cuda")
    for positions in (None, pos, pos.int(), pos[:1]):
        oq, ok = rotary_embed(q, k, cos, sin, positions=positions, layout=layout)
        p = torch.arange(S, device="cuda").expand(B, S) if positions is None else positions.long().expand(B, S)
        pairs = [(q, oq)] + ([(k, ok)] if Hk else [])
        for x, o in pairs:
            ref, mag = ref_rotary(x.detach(), cos[p], sin[p], layout)
            check(o.detach(), ref, 2 * U32 * mag)
            assert torch.equal(o[..., R:], x[..., R:]) and o.is_contiguous()
        assert Hk or ok is None
    dq, dk = _randn(g, B, S, H, D).to(dtype), _randn(g, B, S, Hk, D).to(dtype)
    grads = torch.autograd.grad([o for _, o in pairs], [x for x, _ in pairs], [dq, dk][:len(pairs)])
    for d, gr in zip((dq, dk), grads):
        ref, mag = ref_rotary(d, cos[p], -sin[p], layout)
        check(gr, ref, 2 * U32 * mag)


def test_rotary_slices_of_one_projection(cuda):
    """Queries and keys read in place from a [B, S, 3 * H * D] projection, odd offsets too."""
    B, S, H, D = 2, 33, 3, 64
    for off in (0, 1, 2, 4):
        buf = _randn(_gen(off), B, S, 3 * H * D + off).to(torch.bfloat16)
        qkv = buf[..., off:]
        q, k = qkv[..., :H * D].unflatten(-1, (H, D)), qkv[..., H * D:2 * H * D].unflatten(-1, (H, D))
        cos, sin = table(S, D // 2)
        for layout in ("half", "interleaved"):
            a, b = rotary_embed(q, k, cos, sin, layout=layout)
            c, d = rotary_embed(q.contiguous(), k.contiguous(), cos, sin, layout=layout)
            assert torch.equal(a, c) and torch.equal(b, d)
    # transposed heads, a batched table
    x = _randn(_gen(7), B, H, S, D).to(torch.float16).transpose(1, 2)
    ang = _randn(_gen(8), B, S, D // 2)
    o, _ = rotary_embed(x, None, ang.cos(), ang.sin(), layout="half")
    ref, mag = ref_rotary(x, ang.cos(), ang.sin(), "half")
    check(o, ref, 2 * U32 * mag)


def test_rotary_gradient_only_of_keys_and_of_expanded_outputs(cuda):
    q = _randn(_gen(1), 1, 4, 2, 64)
    k = _randn(_gen(2), 1, 4, 1, 64).requires_grad_()
    cos, sin = table(4, 32)
    _, ok = rotary_embed(q, k, cos, sin)
    (dk,) = torch.autograd.grad(ok.sum(), (k,))
    ref, mag = ref_rotary(torch.ones_like(k), cos[None], -sin[None], "interleaved")
    check(dk, ref, 2 * U32 * mag)


def test_second_derivatives(cuda):
    """A rotation's gradient is a rotation and differentiable again; the others refuse."""
    g = _gen(6)
    q = _randn(g, 1, 5, 2, 32).requires_grad_()
    k = _randn(g, 1, 5, 1, 32).requires_grad_()
    d = _randn(g, 1, 5, 2, 32).requires_grad_()
    e = _randn(g, 1, 5, 2, 32)
    cos, sin = table(5, 16)
    o, _ = rotary_embed(q, k, cos, sin, layout="half")
    (gq,) = torch.autograd.grad(o, (q,), d, create_graph=True)
    (gd,) = torch.autograd.grad(gq, (d,), e)
    ref, mag = ref_rotary(e, cos[None], sin[None], "half")
    check(gd, ref, 2 * U32 * mag)
    x = _randn(g, 4, 9, 32).requires_grad_()
    wq, ws = fp8_block_quantize_weight(_randn(g, 16, 32))
    for y in (group_norm_act(x, 4), fp8_block_linear(x, wq, ws)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y.sum(), (x,), create_graph=True)


def test_rotary_shared_key_gradient_through_expanded_heads(cuda):
    """A key head shared by four query heads (expanded view): its gradient is the sum over them."""
    g = _gen(4)
    base = _randn(g, 2, 5, 1, 32).requires_grad_()
    cos, sin = table(5, 16)
    o, _ = rotary_embed(base.expand(2, 5, 4, 32), None, cos, sin, layout="half")
    d = _randn(g, 2, 5, 4, 32)
    (gr,) = torch.autograd.grad(o, (base,), d)
    ref, mag = ref_rotary(d, cos.expand(2, 5, 16), -sin.expand(2, 5, 16), "half")
    check(gr, ref.sum(2, keepdim=True), 6 * U32 * mag.sum(2, keepdim=True))


def test_rotary_bad_positions_read_nothing(cuda):
    x = _randn(_gen(1), 1, 6, 2, 64)
    cos, sin = table(8, 16)
    pos = torch.tensor([[0, 7, 8, -1, 3, 1 << 40]], device="cuda")
    o, _ = rotary_embed(x, None, cos, sin, positions=pos)
    torch.cuda.synchronize()
    assert _lib.device_error_read_clear() == _lib.ZIB_ERR_INVALID_ARG
    bad = torch.tensor([0, 0, 1, 1, 0, 1], device="cuda").bool()
    assert bool(torch.isnan(o[0, bad, :, :32]).all()) and not bool(torch.isnan(o[0, ~bad]).any())
    assert torch.equal(o[..., 32:], x[..., 32:])
    rotary_embed(x, None, cos, sin)
    assert _lib.device_error_read_clear() == 0


def test_rotary_empty(cuda):
    cos, sin = table(4, 16)
    for shape in ((0, 4, 2, 32), (2, 0, 2, 32), (2, 4, 0, 32)):
        o, _ = rotary_embed(torch.empty(shape, device="cuda"), None, cos, sin)
        assert o.shape == shape


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 8.0},
                                     {"type": "yarn", "factor": 8.0, "original_length": 4096},
                                     {"type": "yarn", "factor": 3.0, "original_length": 100, "beta_fast": 8.0,
                                      "beta_slow": 0.5, "attention_factor": 1.25}])
@pytest.mark.parametrize("dim", [2, 62, 64, 128, 130])
def test_rotary_table(cuda, scaling, dim):
    if dim == 2 and scaling and scaling["type"] == "ntk":
        pytest.skip("ntk scaling is refused for dim 2")
    theta = 10000.0
    pos = torch.cat([torch.arange(300), torch.tensor([-5, 131071, 1 << 20, (1 << 31) - 1])]).cuda()
    f = torch.tensor([theta ** (-2.0 * j / dim) for j in range(dim // 2)], dtype=torch.float64, device="cuda")
    m = 1.0
    if scaling:
        fac = scaling["factor"]
        if scaling["type"] == "linear":
            f = f / fac
        elif scaling["type"] == "ntk":
            f = torch.tensor([(theta * fac ** (dim / (dim - 2))) ** (-2.0 * j / dim) for j in range(dim // 2)],
                             dtype=torch.float64, device="cuda")
        else:
            hi, lo = scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0)
            keep = ((scaling["original_length"] * f / (2 * math.pi) - lo) / (hi - lo)).clamp(0, 1)
            f = f * keep + f / fac * (1 - keep)
            m = scaling.get("attention_factor", 0.1 * math.log(fac) + 1)
    ang = pos.double()[:, None] * f
    for p in (pos, pos.int(), pos.repeat_interleave(2)[::2]):
        cos, sin = rotary_table(p, dim, theta=theta, scaling=scaling)
        # the angle in fp64 (a few steps of 2^-53), sincospi within 2 steps, two more fp32 roundings
        extra = 5 * U32 * m + ang.abs() * 2.0 ** -50 * m
        check(cos, m * ang.cos(), extra)
        check(sin, m * ang.sin(), extra)
    cos, _ = rotary_table(300, dim, theta=theta, scaling=scaling)
    assert torch.equal(cos, rotary_table(pos[:300], dim, theta=theta, scaling=scaling)[0])
    assert rotary_table(0, dim)[0].shape == (0, dim // 2)


# --- group norm -----------------------------------------------------------------------------------


def ref_group_norm(x, G, w, b, eps, act, dy=None):
    """fp64 forward (and gradients), with the fp32 error each may carry before its rounding."""
    B, P, C = x.shape
    xd = x.double().view(B, P, G, C // G)
    mean = xd.mean((1, 3), keepdim=True)
    var = ((xd - mean) ** 2).mean((1, 3), keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    h = (xd - mean) * r
    wd = w.double().view(G, -1) if w is not None else torch.ones(G, C // G, dtype=torch.float64, device=x.device)
    bd = b.double().view(G, -1) if b is not None else torch.zeros_like(wd)
    z = h * wd + bd
    # the stored mean and the subtraction are within a step of |x| + |mean|, h takes two more roundings and
    # the error of 1/sqrt, itself within three steps; z two roundings.  The sums behind the statistics add at
    # most 32 values in a row in fp32 (runs, joined in fp64): 31 additions, each within U32 of the run's sum
    # of magnitudes, so the mean may be off by 31 U32 mean|x|, the variance by 34 U32 of itself (two roundings
    # per squared deviation, 31 additions, one multiply-add less), 1/sqrt by half of that
    avg = xd.abs().mean((1, 3), keepdim=True)
    dh = U32 * (2 * (xd.abs() + mean.abs()) * r + 31 * avg * r + (6 + 17) * h.abs())
    dz = dh * wd.abs() + 2 * U32 * (z.abs() + (h * wd).abs() + bd.abs())
    sig = torch.sigmoid(z)
    if act == "silu":
        y = z * sig
        # exp within 2 + 1.2 |z| steps, the sum, the division and the product within 4; slope at most 1.1
        ey = 1.1 * dz + U32 * y.abs() * (12 + 3 * z.abs())
    else:
        y, ey = z, dz
    out = [(y.view(B, P, C), ey.view(B, P, C))]
    if dy is None:
        return out
    d = dy.double().view_as(xd)
    slope = sig * (1 + z * (1 - sig)) if act == "silu" else torch.ones_like(z)
    g = d * slope
    # the slope's own slope is at most 1/2; sigmoid's relative error as above, and 1 - sig, 1 + z(...) roundings
    eg = d.abs() * (0.5 * dz + U32 * ((12 + 3 * z.abs()) * (1 + z.abs()) * sig + 4)) if act == "silu" else U32 * d.abs()
    n = P * (C // G)
    T = 8 + min(P, 4096) / 8  # additions in a row of one thread's fp32 sums, at most
    A, EA = g.sum((0, 1)), (eg + T * U32 * g.abs()).sum((0, 1))
    E, EE = (g * h).sum((0, 1)), (eg * h.abs() + g.abs() * dh + (T + 2) * U32 * (g * h).abs()).sum((0, 1))
    wg = g * wd
    c1, c2 = wg.sum((1, 3), keepdim=True) / n, (wg * h).sum((1, 3), keepdim=True) / n
    ec1 = ((eg + (T + 3) * U32 * g.abs()) * wd.abs()).sum((1, 3), keepdim=True) / n
    ec2 = ((eg * h.abs() + g.abs() * dh + (T + 3) * U32 * (g * h).abs()) * wd.abs()).sum((1, 3), keepdim=True) / n
    dx = r * (wg - c1 - h * c2)
    edx = r * (eg * wd.abs() + ec1 + ec2 * h.abs() + c2.abs() * dh
               + 6 * U32 * (wg.abs() + c1.abs() + (h * c2).abs()))
    out.append((dx.view(B, P, C), edx.view(B, P, C)))
    return out + [(E.view(C), EE.view(C)), (A.view(C), EA.view(C))]


GN_SHAPES = [(1, 1, 32, 4), (2, 5, 8, 1), (1, 391, 96, 32), (2, 64, 320, 32), (3, 77, 100, 4), (1, 1000, 128, 32),
             (2, 333, 512, 32), (1, 50, 2048, 16), (1, 20, 4104, 27), (4, 9, 7, 7), (1, 4097, 64, 64), (2, 257, 36, 9)]


@pytest.mark.parametrize("act", ["silu", "none"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,P,C,G", GN_SHAPES)
def test_group_norm_forward(cuda, act, dtype, B, P, C, G):
    g = _gen(P + C)
    x = (_randn(g, B, P, C) * (0.5 + torch.rand(C, generator=g, device="cuda")) + _randn(g, C)).to(dtype)
    w, b = 1 + 0.2 * _randn(g, C), 0.2 * _randn(g, C)
    for ww, bb in ((w, b), (None, None), (w.to(torch.bfloat16), None), (None, b.half())):
        y = group_norm_act(x, G, ww, bb, eps=1e-5, activation=act)
        (ref, extra), = ref_group_norm(x, G, ww, bb, 1e-5, act)
        check(y, ref, extra)
        assert y.is_contiguous()


@pytest.mark.parametrize("act", ["silu", "none"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,P,C,G", [s for s in GN_SHAPES if s[1] * s[2] // s[3] >= 16])
def test_group_norm_gradients(cuda, act, dtype, B, P, C, G):
    g = _gen(P + C + 1)
    x = (_randn(g, B, P, C) * (0.5 + torch.rand(C, generator=g, device="cuda")) + _randn(g, C)).to(dtype)
    x.requires_grad_()
    w, b = (1 + 0.2 * _randn(g, C)).requires_grad_(), (0.2 * _randn(g, C)).requires_grad_()
    dy = _randn(g, B, P, C).to(dtype)
    y = group_norm_act(x, G, w, b, eps=1e-5, activation=act)
    got = torch.autograd.grad(y, (x, w, b), dy)
    ref = ref_group_norm(x.detach(), G, w.detach(), b.detach(), 1e-5, act, dy)
    for a, (r, e) in zip(got, ref[1:]):
        check(a, r, e)
    # without parameters, and the parameters alone
    x0 = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(group_norm_act(x0, G, eps=1e-5, activation=act), (x0,), dy)
    check(dx, *ref_group_norm(x.detach(), G, None, None, 1e-5, act, dy)[1])
    dw, db = torch.autograd.grad(group_norm_act(x.detach(), G, w, b, eps=1e-5, activation=act), (w, b), dy)
    assert torch.equal(dw, got[1]) and torch.equal(db, got[2])


@pytest.mark.parametrize("shift,dtype", [(300.0, torch.float32), (3e4, torch.float32), (100.0, torch.float16)])
def test_group_norm_mean_far_from_zero_and_outlier_first(cuda, shift, dtype):
    """A mean many spreads from zero, and a first pixel far from the rest: no cancellation in the sums."""
    x = (_randn(_gen(2), 2, 700, 64) + shift).to(dtype)
    x[1, 0] = 6e4
    y = group_norm_act(x, 8, eps=1e-6, activation="none")
    (ref, extra), = ref_group_norm(x, 8, None, None, 1e-6, "none")
    check(y, ref, extra)


def test_group_norm_constant_and_non_finite_groups(cuda):
    x = _randn(_gen(1), 2, 40, 32).half()
    x[0, :, :8] = 3.0
    x[1, 7, 9] = math.inf
    y = group_norm_act(x, 4, activation="none")
    assert bool((y[0, :, :8] == 0).all())
    bad = torch.isnan(y)
    assert bool(bad[1, :, 8:16].all()) and int(bad.sum()) == 40 * 8


def test_group_norm_strides(cuda):
    """A channels-last convolution tensor, a channel slice and a batch-strided view, read in place."""
    g = _gen(11)
    conv = _randn(g, 2, 64, 9, 7).to(torch.bfloat16).contiguous(memory_format=torch.channels_last)
    x = conv.permute(0, 2, 3, 1)
    w, b = _randn(g, 64), _randn(g, 64)
    y = group_norm_act(x, 16, w, b)
    assert y.shape == (2, 9, 7, 64) and torch.equal(y, group_norm_act(x.contiguous(), 16, w, b))
    wide = _randn(g, 4, 50, 99).half()
    for v in (wide[..., 3:67], wide[::2, 5:, 1:65], wide[..., :64], wide.transpose(1, 2)[:, :64]):
        # other strides allow other access widths, which add in another order: each against the formula
        wv = None if v.shape[-1] != 64 else w
        d = _randn(g, *v.shape).half()
        v = v.detach().requires_grad_()
        a = group_norm_act(v, 2, wv, None)
        (da,) = torch.autograd.grad(a, (v,), d)
        ref = ref_group_norm(v.detach(), 2, wv, None, 1e-6, "silu", d)
        check(a.detach(), *ref[0])
        check(da, *ref[1])
    m = GroupNormAct(16, 64, device="cuda")
    assert torch.equal(m(x), group_norm_act(x, 16, m.weight, m.bias))
    # a broadcast upstream gradient
    xs = x.float().requires_grad_()
    (a,) = torch.autograd.grad(group_norm_act(xs, 16).sum(), (xs,))
    (c,) = torch.autograd.grad(group_norm_act(xs, 16), (xs,), torch.ones(2, 9, 7, 64, device="cuda"))
    assert torch.equal(a, c)


def test_group_norm_empty(cuda):
    w = torch.ones(32, device="cuda", requires_grad=True)
    for shape in ((0, 5, 32), (2, 0, 32)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y = group_norm_act(x, 4, w)
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == shape and dx.shape == shape and bool((dw == 0).all())
    assert group_norm_act(torch.ones(3, 32, device="cuda"), 4).shape == (3, 32)


def test_group_norm_gradient_against_differences(cuda):
    g = _gen(21)
    x = _randn(g, 1, 12, 16)
    dy = _randn(g, 1, 12, 16)
    xs = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(group_norm_act(xs, 4, eps=1e-3), (xs,), dy)
    for p, c in ((0, 0), (5, 7), (11, 15)):
        e = 2.0 ** -6
        up, dn = x.clone(), x.clone()
        up[0, p, c] += e
        dn[0, p, c] -= e
        diff = ((group_norm_act(up, 4, eps=1e-3) - group_norm_act(dn, 4, eps=1e-3)).double() * dy).sum() / (2 * e)
        # third-order term (e^2 times a third derivative of order one, times 192 outputs of which few move
        # much) and the rounding of 192 outputs over the step
        assert abs(float(diff - dx[0, p, c])) <= 20 * e * e + 192 * 8 * U32 / e


# --- together -------------------------------------------------------------------------------------


def test_operators_in_a_row_with_gradients(cuda):
    """norm -> block-quantised projection -> rotation of queries and keys -> attention, both directions.

    The reference runs the same chain in fp64 with the operators' own rounded results taken at the
    quantisers (whose outputs are steps), so each gradient is the chain's formula.
    """
    B, H, W, C, heads, D, G = 2, 6, 5, 256, 4, 64, 32
    S = H * W
    g = _gen(31)
    conv = _randn(g, B, C, H, W).to(torch.bfloat16).contiguous(memory_format=torch.channels_last)
    gw, gb = (1 + 0.1 * _randn(g, C)).requires_grad_(), (0.1 * _randn(g, C)).requires_grad_()
    wq, ws = fp8_block_quantize_weight((_randn(g, 3 * heads * D, C) * 0.06).to(torch.bfloat16))
    wt = fp8_block_transpose(wq)
    cos, sin = rotary_table(S, D, theta=256.0)
    x = conv.permute(0, 2, 3, 1).reshape(B, S, C).detach().requires_grad_()
    dq, dk, dv = (_randn(g, B, S, heads, D).to(torch.bfloat16) for _ in range(3))

    n = group_norm_act(x, G, gw, gb)
    qkv = fp8_block_linear(n, wq, ws, w_q_t=wt)
    q, k, v = (t.unflatten(-1, (heads, D)) for t in qkv.chunk(3, -1))
    rq, rk = rotary_embed(q, k, cos, sin, layout="half")
    dx, dgw, dgb, dn, dqkv = torch.autograd.grad([rq, rk, v], [x, gw, gb, n, qkv], [dq, dk, dv])

    y_ref, y_ext = ref_group_norm(x.detach(), G, gw.detach(), gb.detach(), 1e-6, "silu")[0]
    check(n.detach(), y_ref, y_ext)
    ref, mag = product_terms(*ref_rows(n.detach().view(B * S, C)), wq, ws)
    check(qkv.detach().view(B * S, -1), ref, product_extra(mag, C))
    c2, s2 = cos[None].expand(B, -1, -1), sin[None].expand(B, -1, -1)
    for t, o, d, part in ((q, rq, dq, 0), (k, rk, dk, 1)):
        ref, mag = ref_rotary(t.detach(), c2, s2, "half")
        check(o.detach(), ref, 2 * U32 * mag)
        ref, mag = ref_rotary(d, c2, -s2, "half")
        check(dqkv.chunk(3, -1)[part].unflatten(-1, (heads, D)), ref, 2 * U32 * mag)
    assert torch.equal(dqkv.chunk(3, -1)[2].unflatten(-1, (heads, D)), dv)
    ref, mag = product_terms(*ref_rows(dqkv.view(B * S, -1)), wq.t(), ws.t())
    check(dn.view(B * S, C), ref, product_extra(mag, 3 * heads * D))
    grads = ref_group_norm(x.detach(), G, gw.detach(), gb.detach(), 1e-6, "silu", dn)
    for a, (r, e) in zip((dx, dgw, dgb), grads[1:]):
        check(a, r, e)


def test_operators_captured_and_replayed(cuda):
    """Forward and backward in one graph, two graphs replayed by turns: what the eager calls give."""
    g = _gen(41)
    wq, ws = fp8_block_quantize_weight(_randn(g, 384, 256))
    wt = fp8_block_transpose(wq)
    cos, sin = table(40, 32)
    gw, gb = 1 + 0.1 * _randn(g, 256), 0.1 * _randn(g, 256)

    def step(x, d):
        x = x.detach().requires_grad_()
        w = gw.detach().requires_grad_()
        n = group_norm_act(x, 8, w, gb)
        q = fp8_block_linear(n, wq, ws, w_q_t=wt).unflatten(-1, (6, 64))
        o, _ = rotary_embed(q, None, cos, sin, layout="half")
        return (o.detach(), *torch.autograd.grad(o, (x, w), d))

    ins = [(_randn(g, 2, 40, 256).to(torch.bfloat16), _randn(g, 2, 40, 6, 64).to(torch.bfloat16)) for _ in range(4)]
    eager = [step(*i) for i in ins]
    graphs = []
    for k in range(2):
        x, d = ins[k][0].clone(), ins[k][1].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, d)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(x, d)
        graphs.append((gr, x, d, out))
    for rnd in range(2):
        for k, (gr, x, d, out) in enumerate(graphs):
            i = (2 * rnd + k) % 4
            x.copy_(ins[i][0])
            d.copy_(ins[i][1])
        for gr, *_ in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for k, (gr, x, d, out) in enumerate(graphs):
            for a, b in zip(out, eager[(2 * rnd + k) % 4]):
                assert torch.equal(a, b)


def test_operators_from_two_threads(cuda):
    """Calls of different sizes from two host threads on streams of their own, shared memory sizes included."""
    import threading

    g = _gen(61)
    wq, ws = fp8_block_quantize_weight(_randn(g, 192, 6400))
    cos, sin = table(64, 32)
    work = []
    for M, C in ((1, 4096), (2, 256), (64, 6144), (300, 64)):
        x, y = _randn(g, M, 6400).to(torch.bfloat16), _randn(g, 3, 17, C)
        q = _randn(g, 1, 64, 3, 64)
        work.append((x, y, q, fp8_block_linear(x, wq, ws), group_norm_act(y, C), rotary_embed(q, None, cos, sin)[0]))
    torch.cuda.synchronize()
    bad = []

    def go(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for i in range(40):
                x, y, q, a, b, c = work[(k + i) % len(work)]
                r = (fp8_block_linear(x, wq, ws), group_norm_act(y, y.shape[-1]), rotary_embed(q, None, cos, sin)[0])
                s.synchronize()
                if not all(torch.equal(u, v) for u, v in zip(r, (a, b, c))):
                    bad.append((k, i))

    threads = [threading.Thread(target=go, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_offsets_past_32_bits(cuda):
    """Tensors of more than 2^31 elements: their last rows are what a call on those rows alone gives."""
    g = _gen(71)
    S, H, D = 560000, 30, 128
    q = torch.empty(1, S, H, D, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    assert q.numel() > 1 << 31
    cos, sin = table(S, 64)
    o, _ = rotary_embed(q, None, cos, sin, layout="half")
    t, _ = rotary_embed(q[:, -50:], None, cos[-50:], sin[-50:], layout="half")
    assert torch.equal(o[:, -50:], t)
    del o
    # a batch entry of 2^31 values behind another: statistics against torch's in blocks
    x = q.view(2, S // 2 * H, D)[:, :, :64]
    y = group_norm_act(x, 2, activation="none")
    xd = x[1, -4096:].double().view(4096, 2, 32)
    n = x.shape[1] * 32
    mean = sum(b.double().view(-1, 2, 32).sum((0, 2)) for b in x[1].split(1 << 20)) / n
    var = sum(((b.double().view(-1, 2, 32) - mean[:, None]) ** 2).sum((0, 2)) for b in x[1].split(1 << 20)) / n
    ref = ((xd - mean[:, None]) / torch.sqrt(var[:, None] + 1e-6)).view(4096, 64)
    check(y[1, -4096:], ref, 64 * U32 * (ref.abs() + 1))
    del y
    wq, ws = fp8_block_quantize_weight(_randn(g, 1024, 128))
    rows = q.view(-1, D)[: (1 << 21) + 700]
    z = fp8_block_linear(rows, wq, ws)
    assert z.numel() > 1 << 31
    assert torch.equal(z[-300:], fp8_block_linear(rows[-300:].clone(), wq, ws))
    assert _lib.device_error_read_clear() == 0


def test_fp8_block_linear_module(cuda):
    g = _gen(81)
    lin = torch.nn.Linear(300, 200, device="cuda", dtype=torch.bfloat16)
    m = Fp8BlockLinear.from_linear(lin, transposed=True)
    x = _randn(g, 7, 300).to(torch.bfloat16).requires_grad_()
    wq, ws = fp8_block_quantize_weight(lin.weight)
    assert torch.equal(m(x), fp8_block_linear(x, wq, ws, lin.bias))
    m(x).sum().backward()
    assert x.grad is not None and m.bias is lin.bias and bool((lin.bias.grad == 7).all())
    other = Fp8BlockLinear(300, 200, transposed=True, device="cuda")
    other.load_state_dict(m.state_dict())
    assert torch.equal(other(x), m(x))


def test_operators_on_another_stream(cuda):
    g = _gen(51)
    x = _randn(g, 300, 512).to(torch.bfloat16)
    wq, ws = fp8_block_quantize_weight(_randn(g, 256, 512))
    want = fp8_block_linear(group_norm_act(x, 8), wq, ws)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = fp8_block_linear(group_norm_act(x, 8), wq, ws)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("K", [1, 7, 8, 13, 129, 1001])
def test_quantised_rows_leave_what_lies_behind_them(cuda, K):
    """Rows inside a wider buffer: the kernel stores eights where it can, and nothing past a row's end."""
    x = torch.randn(9, K, generator=_gen(K), device="cuda", dtype=torch.float32)
    ld = (K + 7) // 8 * 8 + 16
    buf = torch.full((9, ld), 0x5A, device="cuda", dtype=torch.uint8)
    s = torch.zeros((K + 127) // 128, 9, device="cuda")
    _lib.call("zib_fp8_quant_rows", x.data_ptr(), K, 2, buf.data_ptr(), ld, s.data_ptr(), 1, 9, 9, K,
              torch.cuda.current_stream().cuda_stream)
    rq, rs = ref_rows(x)
    assert same(buf[:, :K].contiguous().view(torch.float8_e4m3fn), rq) and same(s.t(), rs)
    assert (buf[:, K:] == 0x5A).all()


@pytest.mark.parametrize("K,cut", [(1, 3), (15, 1), (129, 2), (1000, 5)])
def test_weights_at_any_address_and_stride(cuda, K, cut):
    x = torch.randn(40, K, generator=_gen(3), device="cuda", dtype=torch.bfloat16)
    w = torch.randn(70, K, generator=_gen(4), device="cuda", dtype=torch.bfloat16)
    qw, sw = fp8_block_quantize_weight(w)
    wide = torch.zeros(70, K + 9, device="cuda", dtype=torch.uint8)
    wide[:, cut:cut + K] = qw.view(torch.uint8)
    view = wide[:, cut:cut + K].view(torch.float8_e4m3fn)
    even = torch.zeros(70, (K + 15) // 16 * 16, device="cuda", dtype=torch.uint8)
    even[:, :K] = qw.view(torch.uint8)
    even = even.view(torch.float8_e4m3fn)[:, :K]
    assert torch.equal(fp8_block_linear(x, view, sw), fp8_block_linear(x, even, sw))


@pytest.mark.parametrize("M,K,N", [(20, 2000, 346), (45, 257, 130), (100, 1024, 40), (257, 4096, 48), (600, 300, 17)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_groups_of_tokens(cuda, M, K, N, dtype):
    """Few weight rows: tokens in groups of 8, the last one ragged."""
    g = _gen(M + N)
    x, w = (_randn(g, M, K)).to(dtype), (_randn(g, N, K) / 8).to(dtype)
    b = _randn(g, N).to(dtype)
    qw, sw = fp8_block_quantize_weight(w)
    qx, sx = fp8_block_quantize(x)
    ref, mag = product_terms(qx, sx, qw, sw)
    check(fp8_block_linear(x, qw, sw, b), ref + b.double(), product_extra(mag, K, b))


@pytest.mark.parametrize("M,K,N", [(600, 4096, 3840), (600, 1024, 1300), (70, 512, 257), (5, 300, 200)])
def test_linear_captured_with_its_gradients(cuda, M, K, N):
    """Each of the linear's kernels in a captured forward and backward pass, replayed on other inputs."""
    g = _gen(M)
    wq, ws = fp8_block_quantize_weight(_randn(g, N, K) / 16)
    b = _randn(g, N).to(torch.bfloat16)
    ins = [(_randn(g, M, K).to(torch.bfloat16), _randn(g, M, N).to(torch.bfloat16)) for _ in range(3)]

    def step(x, d):
        x, c = x.detach().requires_grad_(), b.detach().requires_grad_()
        y = fp8_block_linear(x, wq, ws, c)
        return (y.detach(), *torch.autograd.grad(y, (x, c), d))

    want = [step(*i) for i in ins]
    x, d = ins[0][0].clone(), ins[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, d)
    for i in (1, 2, 0):
        x.copy_(ins[i][0])
        d.copy_(ins[i][1])
        graph.replay()
        assert all(torch.equal(a, e) for a, e in zip(out, want[i]))


# enough tiles and K-blocks that the tensor cores apply the scales where all are powers of two
MANY_BLOCKS = [(600, 4096, 3840), (1030, 6000, 2001)]


def _varied(g, M, K, spread=12):
    """Values whose 128-blocks differ in size by powers of two."""
    e = torch.randint(-spread, spread + 1, (M, -(-K // 128)), generator=g, device="cuda").float()
    return _randn(g, M, K) * torch.exp2(e).repeat_interleave(128, 1)[:, :K]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", MANY_BLOCKS)
def test_linear_of_many_blocks(cuda, dtype, M, K, N):
    g = _gen(K)
    x = _varied(g, M, K, 3).to(dtype)
    w = _varied(g, N, K, 3) / 64
    bias = _randn(g, N).to(dtype) if N % 2 else None
    wq, ws = fp8_block_quantize_weight(w)
    qx, sx = ref_rows(x)
    ref, mag = product_terms(qx, sx, wq, ws)
    check(fp8_block_linear(x, wq, ws, bias), ref if bias is None else ref + bias.double(), product_extra(mag, K, bias))
    # one scale that is no power of two, of another sign, zero
    for bad in (0.7, -1.0, 0.0):
        other = ws.clone()
        other[-1, -1] = bad
        ref, mag = product_terms(qx, sx, wq, other)
        check(fp8_block_linear(x, wq, other), ref, product_extra(mag, K))
    assert _lib.device_error_read_clear() == 0


def test_linear_of_many_blocks_sums_in_32_bits(cuda):
    M, K, N = 600, 4096, 3840
    x = torch.full((M, K), 2.0 ** -6, device="cuda")
    x[:, ::128], x[:, 1::128] = 448.0, -448.0
    x[:, 3], x[:, 260] = 256.0, -256.0
    y = fp8_block_linear(x, torch.ones(N, K, device="cuda").to(torch.float8_e4m3fn), torch.ones(30, 32, device="cuda"))
    assert bool((y == (K - 66) * 2.0 ** -6).all()), float((y - (K - 66) * 2.0 ** -6).abs().max())


@pytest.mark.parametrize("ex,ew", [(-110, 100), (100, -110), (-60, -60), (60, 60), (-110, 0), (0, 100)])
def test_linear_of_many_blocks_far_exponents(cuda, ex, ew):
    M, K, N = 600, 4096, 3840
    g = _gen(5)
    x, w = _randn(g, M, K), _randn(g, N, K)
    wq, ws = fp8_block_quantize_weight(w)
    qx, sx = ref_rows(x)
    ref, mag = product_terms(qx, sx, wq, ws)
    y = fp8_block_linear(x * 2.0 ** ex, wq, ws * 2.0 ** ew)
    # Compared as they are.  With 60 and 60 an output is 2^120 times a sum whose partial sums, in fp32 like it, reach
    # 2^8 = 2^128 / 2^120 where fp32 ends: no partial sum is larger than the sum of magnitudes, so an infinity
    # is right where that times 2^120 is at least 2^128, and nowhere else.
    f = 2.0 ** (ex + ew)
    over = torch.isinf(y) & (mag * f >= 2.0 ** 128)
    check(torch.where(over, torch.zeros_like(y), y), torch.where(over, torch.zeros_like(ref), ref * f),
          product_extra(mag, K) * f)


def test_linear_of_many_blocks_non_finite(cuda):
    M, K, N = 600, 4096, 3840
    g = _gen(6)
    x, w = _randn(g, M, K).to(torch.bfloat16), _randn(g, N, K)
    x[17, 300], x[599, 4095] = math.inf, math.nan
    wq, ws = fp8_block_quantize_weight(w)
    bad = torch.isnan(fp8_block_linear(x, wq, ws))
    assert bool(bad[17].all()) and bool(bad[599].all()) and int(bad.sum()) == 2 * N
    w[200, 5] = math.inf
    wq, ws = fp8_block_quantize_weight(w)
    bad = torch.isnan(fp8_block_linear(x, wq, ws))
    assert bool(bad[:, 128:256].all()) and int(bad.sum()) == 2 * N + 128 * (M - 2)


def test_linear_of_many_blocks_gradients(cuda):
    M, K, N = 640, 4096, 3840
    g = _gen(7)
    x = _randn(g, M, K).to(torch.bfloat16).requires_grad_()
    b = _randn(g, N).to(torch.bfloat16).requires_grad_()
    wq, ws = fp8_block_quantize_weight(_varied(g, N, K, 3) / 64)
    dy = _varied(g, M, N, 3).to(torch.bfloat16)
    dx, db = torch.autograd.grad(fp8_block_linear(x, wq, ws, b), (x, b), dy)
    ref, mag = product_terms(*ref_rows(dy), wq.t(), ws.t())
    check(dx, ref, product_extra(mag, N))
    check(db, dy.double().sum(0), (M + 2) * U32 * dy.double().abs().sum(0))


def test_gradients_of_dual_gradients_are_refused(cuda):
    """Forward over reverse: a tangent of the upstream gradient would be lost."""
    fw = torch.autograd.forward_ad
    g = _gen(91)
    wq, ws = fp8_block_quantize_weight(_randn(g, 32, 64))
    cos, sin = table(4, 32)
    x = _randn(g, 1, 4, 2, 64).requires_grad_()
    for y in (fp8_block_linear(x, wq, ws), group_norm_act(x, 4), rotary_embed(x, None, cos, sin)[0]):
        with fw.dual_level():
            d = fw.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(y, (x,), d)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("off", [1, 2, 3])
def test_rotary_contiguous_tensors_at_odd_offsets(cuda, layout, dtype, off):
    """Queries, keys and upstream gradients that are contiguous but start on any element."""
    B, S, H, D = 2, 5, 3, 32
    g = _gen(off)

    def at_offset(h):
        buf = _randn(g, B * S * h * D + off).to(dtype)[off:].view(B, S, h, D)
        assert buf.is_contiguous() and buf.data_ptr() % 16 == off * buf.element_size() % 16
        return buf

    q, k, dq, dk = (at_offset(h) for h in (H, 1, H, 1))
    cos, sin = table(S, 10)
    q.requires_grad_(), k.requires_grad_()
    outs = rotary_embed(q, k, cos, sin, layout=layout)
    grads = torch.autograd.grad(outs, (q, k), (dq, dk))
    c2, s2 = cos.expand(B, -1, -1), sin.expand(B, -1, -1)
    for x, o, d, gr in zip((q, k), outs, (dq, dk), grads):
        ref, mag = ref_rotary(x.detach(), c2, s2, layout)
        check(o.detach(), ref, 2 * U32 * mag)
        ref, mag = ref_rotary(d, c2, -s2, layout)
        check(gr, ref, 2 * U32 * mag)
    # in the mixed case one of the two alone is copied
    a, b = rotary_embed(q.detach(), k.detach().clone(), cos, sin, layout=layout)
    assert torch.equal(a, outs[0]) and torch.equal(b, outs[1])


@pytest.mark.parametrize("M", [1, 3, 40])
@pytest.mark.parametrize("N,K", [(1, 17), (1, 8), (1, 250), (5, 100), (40, 1000)])
def test_weight_rows_that_end_with_their_storage(cuda, M, N, K):
    """A one-row weight, and padded rows whose last one has nothing behind it."""
    g = _gen(N + K)
    ld = (K + 15) // 16 * 16
    w = torch.empty((N - 1) * ld + K, dtype=torch.float8_e4m3fn, device="cuda").as_strided((N, K), (ld, 1))
    wq, ws = fp8_block_quantize_weight(_randn(g, N, K))
    w.copy_(wq)
    assert w.untyped_storage().nbytes() == (N - 1) * ld + K
    x = _randn(g, M, K).to(torch.bfloat16).requires_grad_()
    y = fp8_block_linear(x, w, ws)
    ref, mag = product_terms(*ref_rows(x.detach()), wq, ws)
    check(y.detach(), ref, product_extra(mag, K))
    d = _randn(g, M, N).to(torch.bfloat16)
    (dx,) = torch.autograd.grad(y, (x,), d)
    ref, mag = product_terms(*ref_rows(d), wq.t(), ws.t())
    check(dx, ref, product_extra(mag, N))
    assert torch.equal(fp8_block_matmul(*fp8_block_quantize(x.detach()), w, ws),
                       fp8_block_matmul(*fp8_block_quantize(x.detach()), wq, ws))


@pytest.mark.parametrize("K,N", [(300, 200), (129, 70), (64, 1)])
def test_fp8_block_linear_module_moved_and_loaded(cuda, K, N):
    """To the host and back, and into a layer of the constructor's: the same results from aligned rows."""
    g = _gen(K)
    lin = torch.nn.Linear(K, N, device="cuda", dtype=torch.bfloat16)
    m = Fp8BlockLinear.from_linear(lin, transposed=True)
    x = _randn(g, 7, K).to(torch.bfloat16).requires_grad_()
    y = m(x)
    (dx,) = torch.autograd.grad(y.sum(), (x,))
    other = Fp8BlockLinear(K, N, transposed=True, device="cuda")
    other.load_state_dict(m.state_dict())
    for n in (other, m.cpu().cuda()):
        assert all(t.stride(0) % 16 == 0 and t.stride(1) == 1 for t in (n.w_q, n.w_q_t))
        assert torch.equal(n(x), y) and torch.equal(torch.autograd.grad(n(x).sum(), (x,))[0], dx)


@pytest.mark.parametrize("B", [65535, 65536, 70001, 131072])
def test_group_norm_of_many_batch_entries(cuda, B):
    """A matrix [rows, C]: its rows are the batch entries."""
    g = _gen(B)
    C, G = 64, 4
    x, dy = _randn(g, B, C).to(torch.bfloat16).requires_grad_(), _randn(g, B, C).to(torch.bfloat16)
    w, b = (1 + 0.2 * _randn(g, C)).requires_grad_(), (0.2 * _randn(g, C)).requires_grad_()
    y = group_norm_act(x, G, w, b)
    got = torch.autograd.grad(y, (x, w, b), dy)
    ref = ref_group_norm(x.detach()[:, None], G, w.detach(), b.detach(), 1e-6, "silu", dy[:, None])
    check(y.detach()[:, None], *ref[0])
    check(got[0][:, None], *ref[1])
    for a, r in zip(got[1:], ref[2:]):
        check(a, *r)


@pytest.mark.parametrize("G", [4, 128])
def test_group_norm_of_many_batch_entries_in_two_passes(cuda, G):
    """One image seen by 65537 batch entries (stride 0), too large for the one-launch form."""
    g = _gen(G)
    B, P, C = 65537, 1030, 128
    one, d = _randn(g, 1, P, C).to(torch.bfloat16), _randn(g, 1, P, C).to(torch.bfloat16)
    w, b = (1 + 0.2 * _randn(g, C)).requires_grad_(), (0.2 * _randn(g, C)).requires_grad_()
    x = one.expand(B, P, C).detach().requires_grad_()
    y = group_norm_act(x, G, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), d.expand(B, P, C))
    y = y.detach()
    ref = ref_group_norm(one, G, w.detach(), b.detach(), 1e-6, "silu", d)
    check(y[:1], *ref[0])
    check(dx[:1], *ref[1])
    for part in (y, dx):
        assert all(bool((t == part[:1]).all()) for t in part.split(4096))
    # B equal terms for each of one entry's, joined in fp64
    check(dw, ref[2][0] * B, ref[2][1] * B)
    check(db, ref[3][0] * B, ref[3][1] * B)


def test_group_norm_parameter_gradients_of_long_sums(cuda):
    """Many pixels to a cluster, all terms of one sign: each addition in 32 bits errs the same way."""
    g = _gen(101)
    B, P, C, G = 30, 1 << 17, 1024, 32
    one = _randn(g, 1, P, C)
    d = (1 / 3 + torch.arange(C, device="cuda") / 7).expand(1, P, C)
    w, b = torch.ones(C, device="cuda", requires_grad=True), torch.zeros(C, device="cuda", requires_grad=True)
    y = group_norm_act(one.expand(B, P, C), G, w, b, activation="none")
    dw, db = torch.autograd.grad(y, (w, b), d.expand(B, P, C))
    # 511 additions of a thread's run of 512 at most, one rounding of the CTA's sum, seven additions of the cluster's
    n = 511 + 1 + 7
    check(db, B * P * d[0, 0].double(), n * U32 * B * P * d[0, 0].double())
    xd = one.double().view(P, G, C // G)
    mean = xd.mean((0, 2), keepdim=True)
    r = 1 / torch.sqrt(((xd - mean) ** 2).mean((0, 2), keepdim=True) + 1e-6)
    h = ((xd - mean) * r).view(P, C)
    # h as in ref_group_norm (the subtraction, the statistics' own error), one more step for the multiply-add
    dh = U32 * (2 * (one[0].double().abs() + mean.abs().max()) * r.max() + 31 * r.max() + 23 * h.abs())
    gh = d[0].double() * h
    check(dw, B * gh.sum(0), B * (d[0].double() * dh + (n + 1) * U32 * gh.abs()).sum(0))


@pytest.mark.parametrize("dim,theta", [(128, 10000.0), (128, 500000.0), (62, 256.0), (64, 1e6)])
def test_rotary_table_keeps_small_angles(cuda, dim, theta):
    """Relative to each value: slow frequencies at early positions have small sines."""
    pos = torch.cat([torch.arange(-40, 300), torch.tensor([1000, 4095, 131071, (1 << 31) - 1])]).cuda()
    f = torch.tensor([theta ** (-2.0 * j / dim) for j in range(dim // 2)], dtype=torch.float64, device="cuda")
    p = pos.double()[:, None]
    ang = p * f
    cos, sin = rotary_table(pos, dim, theta=theta)
    for got, ref in ((cos, ang.cos()), (sin, ang.sin())):
        # the rest of the angle: two conversions joined in one multiply-add, the constant and the product, four
        # roundings; the series' last step, its terms before (a tenth of it, four roundings) and what it leaves out
        # (2e-9 of an eighth of a turn, a thirtieth of a step), the factor: seven steps of the value.  The angle's
        # own error: 2^-55 turns a position for its fp64 frequency, 2^-64 for its fixed point, and the
        # reference's, three steps of 2^-53
        check(got, ref, 7 * U32 * ref.abs() + p.abs() * 2 * math.pi * (2.0 ** -55 + 2.0 ** -64) + ang.abs() * 2.0 ** -51)
    s = sin[pos == 1][0]
    small = f < 1e-3
    if bool(small.any()):
        assert bool(((s.double() - f.sin()).abs() <= 8 * U32 * f)[small].all())


# --- several tiles to a pair of CTAs ------------------------------------------------------------------

# 74 pairs.  By the launch rule: 360 tiles of 256 x 192 where the tensor cores apply the scales and, for other
# scales, 270 of 256 x 256; 143 of 256 x 128
SEVERAL_TILES = [(4608, 2048, 3840), (4500, 2000, 3701)]
SEVERAL_SLIM_TILES = [(3328, 1024, 1408), (3300, 1000, 1399)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SEVERAL_TILES)
def test_linear_of_several_tiles_to_a_pair(cuda, dtype, M, K, N):
    """Accumulators, stages, scales and the bias' copy used again by a pair's next tiles."""
    g = _gen(M + K)
    x = _varied(g, M, K, 3).to(dtype)
    wq, ws = fp8_block_quantize_weight(_varied(g, N, K, 3) / 64)
    bias = (_randn(g, N) * 30).to(dtype)
    qx, sx = ref_rows(x)
    ref, mag = product_terms(qx, sx, wq, ws)
    check(fp8_block_linear(x, wq, ws, bias), ref + bias.double(), product_extra(mag, K, bias))
    check(fp8_block_linear(x, wq, ws), ref, product_extra(mag, K))
    other = ws.clone()
    other[-1, -1] = 0.7  # no power of two: the second launch
    ref, mag = product_terms(qx, sx, wq, other)
    check(fp8_block_linear(x, wq, other, bias), ref + bias.double(), product_extra(mag, K, bias))
    assert _lib.device_error_read_clear() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SEVERAL_TILES + SEVERAL_SLIM_TILES)
def test_matmul_of_several_tiles_to_a_pair(cuda, dtype, M, K, N):
    g = _gen(M + K + 1)
    xq, sx = fp8_block_quantize(_varied(g, M, K, 3))
    wq, sw = fp8_block_quantize_weight(_varied(g, N, K, 3) / 64)
    bias = (_randn(g, N) * 30).to(dtype)
    sx = sx * (0.5 + torch.rand(sx.shape, generator=g, device="cuda"))
    ref, mag = product_terms(xq, sx, wq, sw)
    # the product of the two scales is rounded once more where they are no powers of two
    y = fp8_block_matmul(xq, sx, wq, sw, bias, out_dtype=dtype)
    check(y, ref + bias.double(), product_extra(mag, K, bias))
    assert _lib.device_error_read_clear() == 0


def test_linear_gradients_of_several_tiles_to_a_pair(cuda):
    M, K, N = 4608, 3840, 2048
    g = _gen(103)
    x = _randn(g, M, K).to(torch.bfloat16).requires_grad_()
    b = _randn(g, N).to(torch.bfloat16).requires_grad_()
    wq, ws = fp8_block_quantize_weight(_varied(g, N, K, 3) / 64)
    dy = _varied(g, M, N, 3).to(torch.bfloat16)
    want = product_terms(*ref_rows(dy), wq.t(), ws.t())
    for wt in (None, fp8_block_transpose(wq)):
        dx, db = torch.autograd.grad(fp8_block_linear(x, wq, ws, b, w_q_t=wt), (x, b), dy)
        check(dx, want[0], product_extra(want[1], N))
        check(db, dy.double().sum(0), (M + 2) * U32 * dy.double().abs().sum(0))


# --- what the sums hold -------------------------------------------------------------------------------


@pytest.mark.parametrize("M,K,N,quantised", [(600, 4096, 3840, False), (600, 4096, 3840, True), (600, 4096, 128, True),
                                             (8, 4096, 3840, False), (2, 4096, 256, False), (200, 4096, 128, False)])
@pytest.mark.parametrize("at", [1, 31, 32, 64, 127, 128])
def test_sums_hold_24_bits(cuda, M, K, N, quantised, at):
    """2^16 and a term of 2^-7 in the same step, in another one of its block, or 31 of them in other blocks: every
    partial sum is a multiple of 2^-7 below 2^17, so exact in 24 bits, in any order."""
    x = torch.zeros(M, K, device="cuda")
    x[:, 0] = 256.0
    x[:, 2] = 448.0  # the block's scale is 1; its weights are 0
    x[:, at::128] = 2.0 ** -6 if at < 128 else 0.0
    if at == 128:
        x[:, 128::128] = 2.0 ** -6
        x[:, 130::128] = 448.0
    w = torch.zeros(N, K, device="cuda")
    w[:, 0] = 256.0
    w[:, at::128] = 2.0 ** -1
    if at < 128:
        w[:, 128:] = 0.0
    wq, ws = w.to(torch.float8_e4m3fn), torch.ones(-(-N // 128), K // 128, device="cuda")
    q, s = fp8_block_quantize(x)
    assert bool((s[:, 0] == 1).all()) and same(q, x / s.repeat_interleave(128, 1))
    y = fp8_block_matmul(q, s, wq, ws, out_dtype=torch.float32) if quantised else fp8_block_linear(x, wq, ws)
    assert bool((y == 65536.0 + (1 if at < 128 else 31) * 2.0 ** -7).all()), float(y.flatten()[0] - 65536.0)


@pytest.mark.parametrize("ex,ew", [(50, 60), (60, 50), (-50, -60), (100, 10)])
def test_linear_of_many_blocks_far_exponents_within_range(cuda, ex, ew):
    """The sum of magnitudes times 2^(ex + ew) stays below 2^128, so no partial sum may be infinite."""
    M, K, N = 600, 4096, 3840
    g = _gen(15)
    x, w = _randn(g, M, K), _randn(g, N, K)
    wq, ws = fp8_block_quantize_weight(w)
    ref, mag = product_terms(*ref_rows(x), wq, ws)
    f = 2.0 ** (ex + ew)
    assert float(mag.max()) * f < 2.0 ** 127
    y = fp8_block_linear(x * 2.0 ** ex, wq, ws * 2.0 ** ew)
    assert bool(torch.isfinite(y).all())
    check(y, ref * f, product_extra(mag, K) * f)


# --- group norm: many groups in two passes, and each parameter alone ------------------------------------

MANY_GROUPS = [(2, 900, 768, 96), (1, 700, 1024, 1024), (3, 1100, 325, 65), (1, 2000, 1000, 125)]


@pytest.mark.parametrize("act", ["silu", "none"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,P,C,G", MANY_GROUPS)
def test_group_norm_of_many_groups(cuda, act, dtype, B, P, C, G):
    g = _gen(P + C)
    x = (_randn(g, B, P, C) * (0.5 + torch.rand(C, generator=g, device="cuda")) + _randn(g, C)).to(dtype)
    x.requires_grad_()
    w, b = (1 + 0.2 * _randn(g, C)).requires_grad_(), (0.2 * _randn(g, C)).requires_grad_()
    dy = _randn(g, B, P, C).to(dtype)
    y = group_norm_act(x, G, w, b, eps=1e-5, activation=act)
    ref = ref_group_norm(x.detach(), G, w.detach(), b.detach(), 1e-5, act, dy)
    for a, (r, e) in zip((y.detach(), *torch.autograd.grad(y, (x, w, b), dy)), ref):
        check(a, r, e)


@pytest.mark.parametrize("pdtype", TYPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,P,C,G", [(2, 64, 320, 32), (2, 900, 768, 96), (1, 4097, 64, 4)])
def test_group_norm_gradients_of_each_parameter(cuda, pdtype, dtype, B, P, C, G):
    """Weights and biases of each type, together, one of them given, one of them wanted."""
    g = _gen(P + C + 7)
    x = (_randn(g, B, P, C) + _randn(g, C)).to(dtype)
    w, b = (1 + 0.2 * _randn(g, C)).to(pdtype), (0.2 * _randn(g, C)).to(pdtype)
    dy = _randn(g, B, P, C).to(dtype)
    for has_w, has_b in ((True, True), (True, False), (False, True)):
        ref = ref_group_norm(x, G, w if has_w else None, b if has_b else None, 1e-5, "silu", dy)
        for want_x, want_w, want_b in ((True, has_w, has_b), (False, has_w, False), (False, False, has_b)):
            if not (want_x or want_w or want_b):
                continue
            xx = x.detach().requires_grad_(want_x)
            ww = w.detach().requires_grad_(want_w) if has_w else None
            bb = b.detach().requires_grad_(want_b) if has_b else None
            y = group_norm_act(xx, G, ww, bb, eps=1e-5)
            leaves = [(t, r) for t, wanted, r in ((xx, want_x, ref[1]), (ww, want_w, ref[2]), (bb, want_b, ref[3])) if wanted]
            for a, (t, r) in zip(torch.autograd.grad(y, [t for t, _ in leaves], dy), leaves):
                assert a.dtype == t.dtype
                check(a, *r)


def test_views_that_read_as_negatives_are_refused(cuda):
    """Such as the imaginary part of a conjugate: memory holds the other sign."""
    g = _gen(105)
    x, wq, ws = _randn(g, 4, 64), *fp8_block_quantize_weight(_randn(g, 8, 64))
    z = torch.complex(_randn(g, 1, 1), _randn(g, 1, 1)).conj()
    neg = torch._neg_view
    c = _randn(g, 4, 8)
    q = _randn(g, 1, 4, 2, 16)
    for call in (lambda: fp8_block_linear(x, wq, z.imag), lambda: fp8_block_linear(neg(x), wq, ws),
                 lambda: fp8_block_quantize(neg(x)), lambda: fp8_block_quantize_weight(neg(x)),
                 lambda: rotary_embed(neg(q), None, c, c), lambda: rotary_embed(q, neg(q), c, c),
                 lambda: rotary_embed(q, None, c, neg(c)), lambda: group_norm_act(neg(x), 4),
                 lambda: group_norm_act(x, 4, neg(torch.ones(64, device="cuda")))):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()
    # upstream gradients are resolved
    xs = x.detach().requires_grad_()
    for y in (fp8_block_linear(xs, wq, ws), group_norm_act(xs, 4), rotary_embed(xs.view(1, 4, 4, 16), None, c, c)[0]):
        d = _randn(g, *y.shape)
        a, b = (torch.autograd.grad(y, (xs,), t, retain_graph=True)[0] for t in (neg(d), -d))
        assert torch.equal(a, b)


@pytest.mark.parametrize("laid_out", [False, True])
def test_linear_keeps_no_copy_of_the_weight(cuda, laid_out):
    """A weight whose rows are copied to aligned ones: the copy ends with the call, not with the backward pass."""
    g = _gen(107)
    M, K, N = 4, 2001, 1000
    wq, ws = fp8_block_quantize_weight(_randn(g, N, K))
    w = wq.contiguous()
    wt = fp8_block_transpose(wq) if laid_out else None
    x = _randn(g, M, K).to(torch.bfloat16).requires_grad_()
    y = fp8_block_linear(x, w, ws, w_q_t=wt)
    del y
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = fp8_block_linear(x, w, ws, w_q_t=wt)
    assert torch.cuda.memory_allocated() - before < 1 << 20 < w.numel()
    d = _randn(g, M, N).to(torch.bfloat16)
    (dx,) = torch.autograd.grad(y, (x,), d)
    ref, mag = product_terms(*ref_rows(d), wq.t(), ws.t())
    check(dx, ref, product_extra(mag, N))
