"""What the block-scaled 8-bit products, rotary positions and group normalisation refuse, before any launch."""

import math

import pytest
import torch

from zimage_b200 import (Fp8BlockLinear, GroupNormAct, _lib, fp8_block_linear, fp8_block_matmul, fp8_block_quantize,
                         fp8_block_quantize_weight, fp8_block_transpose, group_norm_act, rotary_embed, rotary_table)

E4M3 = torch.float8_e4m3fn
INV = _lib.ZIB_ERR_INVALID_ARG


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 128)
    with pytest.raises(ValueError, match="CUDA"):
        fp8_block_quantize(x)
    with pytest.raises(ValueError, match="CUDA"):
        fp8_block_quantize_weight(x)
    with pytest.raises(ValueError, match="CUDA"):
        fp8_block_transpose(x.to(E4M3))
    with pytest.raises(ValueError, match="CUDA"):
        fp8_block_linear(x, torch.zeros(64, 128).to(E4M3), torch.ones(1, 1))
    with pytest.raises(ValueError, match="CUDA"):
        group_norm_act(x, 4)
    with pytest.raises(ValueError, match="CUDA"):
        rotary_embed(torch.zeros(1, 2, 1, 8), None, torch.ones(2, 4), torch.ones(2, 4))
    with pytest.raises(ValueError, match="CUDA"):
        rotary_table(torch.arange(4), 8)


def test_fp8_shapes_and_types():
    x, w, s = torch.zeros(3, 200), torch.zeros(130, 200).to(E4M3), torch.ones(2, 2)
    for bad in (dict(w_q=w.float()), dict(w_q=w[:, :128]), dict(w_scale=s[:1]), dict(w_scale=s.double()),
                dict(bias=torch.zeros(129)), dict(bias=torch.zeros(130).half()), dict(w_q_t=w),
                dict(w_q_t=torch.zeros(200, 130))):
        kw = {"w_q": w, "w_scale": s, **bad}
        with pytest.raises(ValueError):
            fp8_block_linear(x, **kw)
    with pytest.raises(ValueError, match="bfloat16, float16 or float32"):
        fp8_block_linear(x.double(), w, s)
    with pytest.raises(ValueError):
        fp8_block_quantize(torch.zeros(4, 0))
    with pytest.raises(ValueError):
        fp8_block_quantize(torch.zeros(()))
    with pytest.raises(ValueError):
        fp8_block_quantize_weight(torch.zeros(2, 3, 4))
    with pytest.raises(ValueError):
        fp8_block_transpose(torch.zeros(4, 4))
    xq, xs = x.to(E4M3), torch.ones(3, 2)
    for args in ((x, xs, w, s), (xq, xs[:2], w, s), (xq, xs.half(), w, s), (xq, xs, w, s[:1])):
        with pytest.raises(ValueError):
            fp8_block_matmul(*args)
    with pytest.raises(ValueError, match="out_dtype"):
        fp8_block_matmul(xq, xs, w, s, out_dtype=torch.float64)


def test_rotary_shapes_and_types():
    q, c = torch.zeros(2, 3, 4, 16), torch.ones(5, 8)
    bad = [
        (q[0], None, c, c, {}), (q, q[:1], c, c, {}), (q, q.half(), c, c, {}), (q, q[..., :8], c, c, {}),
        (q, None, c, c[:4], {}), (q, None, c.double(), c.double(), {}), (q, None, c[:2], c[:2], {}),
        (q, None, torch.ones(5, 9), torch.ones(5, 9), {}), (q, None, torch.ones(5, 0), torch.ones(5, 0), {}),
        (q, None, torch.ones(3, 5, 8), torch.ones(3, 5, 8), {}), (q, None, c, c, {"layout": "other"}),
        (q, None, c, c, {"positions": torch.zeros(2, 3)}),
        (q, None, c, c, {"positions": torch.zeros(2, 4, dtype=torch.long)}),
        (q, None, c[:0], c[:0], {"positions": torch.zeros(2, 3, dtype=torch.long)}),
        (q.double(), None, c, c, {}), (torch.zeros(1, 1, 1, 15), None, c[:, :7], c[:, :7], {}),
        (torch.zeros(1, 1, 1, 2048), None, c, c, {}),
    ]
    for a, b, cos, sin, kw in bad:
        with pytest.raises(ValueError):
            rotary_embed(a, b, cos, sin, **kw)


def test_rotary_table_arguments():
    for dim in (0, 3, -2, 8.0):
        with pytest.raises(ValueError):
            rotary_table(4, dim)
    for sc in ({"type": "other"}, {"factor": 2.0}, {"type": "linear", "factor": 0.5}, {"type": "ntk", "factor": math.nan},
               {"type": "yarn", "factor": 2.0}, {"type": "linear", "factor": 2.0, "extra": 1},
               {"type": "yarn", "factor": 2.0, "original_length": 10, "beta_fast": 1.0, "beta_slow": 2.0},
               {"type": "yarn", "factor": 2.0, "original_length": 10, "attention_factor": 0.0}):
        with pytest.raises(ValueError):
            rotary_table(torch.arange(4), 8, scaling=sc)
    with pytest.raises(ValueError):
        rotary_table(torch.zeros(4), 8)
    with pytest.raises(ValueError):
        rotary_table(torch.zeros(2, 2, dtype=torch.long), 8)


def test_group_norm_arguments():
    x = torch.zeros(2, 5, 12)
    for args, kw in (((x, 5), {}), ((x, 0), {}), ((x[0, 0], 4), {}), ((x.double(), 4), {}),
                     ((x, 4, torch.ones(11)), {}), ((x, 4, torch.ones(12).double()), {}),
                     ((x, 4, torch.ones(12), torch.ones(12).half()), {}), ((x, 4), {"activation": "other"}),
                     ((x, 4), {"eps": -1.0}), ((x, 4), {"eps": math.nan})):
        with pytest.raises(ValueError):
            group_norm_act(*args, **kw)
    with pytest.raises(RuntimeError, match="at most"):
        group_norm_act(torch.zeros(1, 1, 8200), 8)
    with pytest.raises(ValueError):
        GroupNormAct(5, 12)
    with pytest.raises(ValueError):
        GroupNormAct(4, 12, activation="other")


def test_c_entries_validate_on_the_host():
    lib = _lib.load()
    # null operands, unknown types, impossible shapes: an error code, no launch
    assert lib.zib_fp8_quant_rows(None, 128, 0, None, 128, None, 1, 1, 4, 128, None) == INV
    assert lib.zib_fp8_quant_rows(16, 128, 7, 16, 128, 16, 1, 1, 4, 128, None) == INV
    assert lib.zib_fp8_quant_rows(16, 64, 0, 16, 128, 16, 1, 1, 4, 128, None) == INV
    assert lib.zib_fp8_quant_blocks(16, 128, 0, 16, 128, 16, 1, 1, 0, 128, None) == INV
    assert lib.zib_fp8_block_gemm(16, 128, 16, 1, 1, 16, 128, 16, 1, 1, None, 16, 8, 9, 4, 8, 128, None) == INV
    assert lib.zib_fp8_block_gemm(16, 120, 16, 1, 1, 16, 128, 16, 1, 1, None, 16, 8, 0, 4, 8, 120, None) == \
        _lib.ZIB_ERR_ALIGNMENT
    assert lib.zib_fp8_block_gemm(24, 128, 16, 1, 1, 16, 128, 16, 1, 1, None, 16, 8, 0, 4, 8, 128, None) == \
        _lib.ZIB_ERR_ALIGNMENT
    assert lib.zib_fp8_block_gemm(16, 1 << 31, 16, 1, 1, 16, 1 << 31, 16, 1, 1, None, 16, 8, 0, 4, 8, 1 << 31, None) \
        == _lib.ZIB_ERR_TOO_LARGE
    assert lib.zib_fp8_block_gemm(None, 128, None, 1, 1, None, 128, None, 1, 1, None, None, 8, 0, 0, 8, 128, None) == 0
    assert lib.zib_fp8_block_linear(16, 64, 0, 16, 128, 16, 1, 1, None, 16, 8, None, None, 0, 4, 8, 128, None) == INV
    assert lib.zib_fp8_block_linear(16, 128, 0, 16, 120, 16, 1, 1, None, 16, 8, None, None, 0, 4, 8, 120, None) == \
        _lib.ZIB_ERR_ALIGNMENT
    assert lib.zib_fp8_block_linear(16, 128, 0, 16, 128, 16, 1, 1, None, 16, 8, None, 128, 64, 40, 8, 128, None) == INV
    assert lib.zib_fp8_block_linear(None, 128, 0, None, 128, None, 1, 1, None, None, 8, None, None, 0, 0, 8, 128, None) == 0
    assert lib.zib_fp8_block_linear_scratch(0, 128, 0) == 0
    assert lib.zib_fp8_block_linear_scratch(1, 128, 0) == 0
    assert lib.zib_fp8_block_linear_scratch(40, 130, 0) >= 40 * 144 + 2 * 40 * 4
    assert lib.zib_fp8_block_linear_scratch(40, 130, 1) >= 40 * 144 + 2 * 40 * 4 + 130 * 4
    assert lib.zib_fp8_transpose(None, 8, None, 8, 8, 8, None) == INV
    assert lib.zib_col_sum(16, 8, 0, 16, 16, 4, 4, 8, None) == INV
    rot = [16, 0, 0, 0, 16, 1, None, 0, 0, 0, None, 0]
    tab = [16, 16, 0, 4, 8, None, 0, 0, 0]
    assert lib.zib_rotary(*rot, 5, *tab, 1, 1, 8, 8, 0, 0, None) == INV
    assert lib.zib_rotary(*rot, 0, *tab, 1, 1, 8, 6 + 1, 0, 0, None) == INV
    assert lib.zib_rotary(*rot, 0, *tab, 1, 1, 8, 10, 0, 0, None) == INV
    assert lib.zib_rotary(*rot, 0, *tab, 1, 9, 8, 8, 0, 0, None) == INV  # 9 tokens, 8 rows
    assert lib.zib_rotary(*rot, 0, *tab, 0, 9, 8, 8, 0, 0, None) == 0
    assert lib.zib_rotary(17, *rot[1:], 0, *tab, 1, 1, 8, 8, 0, 0, None) == _lib.ZIB_ERR_ALIGNMENT
    assert lib.zib_rotary_table(None, 0, 0, 0, 4, 7, 1e4, 0, 1.0, 0.0, 32.0, 1.0, 1.0, 16, 16, None) == INV
    assert lib.zib_rotary_table(None, 0, 0, 0, 4, 8, -1.0, 0, 1.0, 0.0, 32.0, 1.0, 1.0, 16, 16, None) == INV
    assert lib.zib_rotary_table(None, 0, 0, 0, 4, 2, 1e4, 2, 2.0, 0.0, 32.0, 1.0, 1.0, 16, 16, None) == INV
    assert lib.zib_rotary_table(None, 0, 0, 0, 4, 8, 1e4, 3, 2.0, 0.0, 32.0, 1.0, 1.0, 16, 16, None) == INV
    gn = [16, 0, 0, 16, None, None, 0, 16, 16, 16]
    assert lib.zib_group_norm(*gn, 1 << 20, 1, 4, 12, 5, 0, 1e-6, 1, None) == INV
    assert lib.zib_group_norm(*gn, 1 << 20, 1, 4, 12, 4, 0, 1e-6, 9, None) == INV
    assert lib.zib_group_norm(*gn, 0, 1, 4, 12, 4, 0, 1e-6, 1, None) == INV  # workspace
    assert lib.zib_group_norm(*gn, 1 << 40, 1, 4, 1 << 14, 4, 0, 1e-6, 1, None) == _lib.ZIB_ERR_TOO_LARGE
    assert lib.zib_group_norm(*gn, 0, 0, 4, 12, 4, 0, 1e-6, 1, None) == 0
    assert lib.zib_group_norm_workspace(0, 4, 12, 4, 0) == 0
    assert lib.zib_group_norm_workspace(2, 400, 12, 4, 1) > 0


@pytest.mark.parametrize("cast", [lambda m: m.to(torch.float16), lambda m: m.half(), lambda m: m.double(),
                                  lambda m: torch.nn.Sequential(m).float()[0]])
def test_fp8_block_linear_keeps_its_weight_through_casts(cast):
    m = Fp8BlockLinear(130, 70, transposed=True)
    m.w_q.view(torch.uint8).random_(0, 100)
    q, s = m.w_q.clone(), m.w_scale.clone()
    want = cast(torch.nn.Linear(1, 1)).bias.dtype
    m = cast(m)
    assert m.bias.dtype == want
    assert m.w_q.dtype == m.w_q_t.dtype == torch.float8_e4m3fn and m.w_scale.dtype == torch.float32
    assert torch.equal(m.w_q.view(torch.uint8), q.view(torch.uint8)) and torch.equal(m.w_scale, s)


def test_forward_mode_derivatives_are_refused():
    """A dual tensor that requires no gradient: the output would have no tangent, and nothing would say so."""
    fw = torch.autograd.forward_ad
    x, c = torch.ones(1, 2, 2, 8), torch.ones(2, 4)
    w, s = torch.zeros(4, 8).to(E4M3), torch.ones(1, 1)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: fp8_block_linear(dual(x), w, s), lambda: fp8_block_linear(x, w, s, dual(torch.zeros(4))),
                     lambda: fp8_block_linear(x, w, dual(s)), lambda: rotary_embed(dual(x), None, c, c),
                     lambda: rotary_embed(x, dual(x), c, c), lambda: rotary_embed(x, None, c, dual(c)),
                     lambda: group_norm_act(dual(x), 2), lambda: group_norm_act(x, 2, dual(torch.ones(8))),
                     lambda: group_norm_act(x, 2, None, dual(torch.ones(8)))):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
            with fw._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="CUDA"):
                call()


def test_tracing_is_refused():
    """A trace would hold the allocation of the output without the kernel that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x, c = torch.ones(1, 2, 2, 8), torch.ones(2, 4)
    w, s = torch.zeros(4, 8).to(E4M3), torch.ones(1, 1)
    xq, xs = torch.zeros(3, 8).to(E4M3), torch.ones(3, 1)
    for call in (lambda t: fp8_block_quantize(t), lambda t: fp8_block_quantize_weight(t[0, 0]),
                 lambda t: fp8_block_transpose(w), lambda t: fp8_block_matmul(xq, xs, w, s),
                 lambda t: fp8_block_linear(t, w, s), lambda t: rotary_embed(t, None, c, c)[0],
                 lambda t: rotary_table(torch.arange(4), 8), lambda t: rotary_table(4, 8),
                 lambda t: group_norm_act(t, 2), Fp8BlockLinear(8, 4), GroupNormAct(2, 8)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, (x,))
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(call)(x)


@pytest.mark.parametrize("K,N", [(130, 70), (64, 33), (17, 1), (1, 17), (128, 256)])
def test_fp8_block_linear_keeps_its_rows_aligned(K, N):
    """Through the constructor, loading (copied and assigned), casts, moves, copies and files."""
    import copy
    import io

    def check(m):
        for t in (m.w_q, m.w_q_t):
            assert t.dtype == E4M3 and t.stride(0) % 16 == 0 and t.stride(1) == 1
            assert t.device.type == "meta" or t.data_ptr() % 16 == 0
        return m

    dense = {"w_q": torch.randint(0, 100, (N, K), dtype=torch.uint8).view(E4M3), "w_scale": torch.rand(-(-N // 128), -(-K // 128)),
             "bias": torch.zeros(N, dtype=torch.bfloat16)}
    dense["w_q_t"] = dense["w_q"].t().contiguous()
    check(Fp8BlockLinear(K, N, transposed=True, device="meta"))
    new = lambda: check(Fp8BlockLinear(K, N, transposed=True))  # noqa: E731
    made = []
    for assign in (False, True):
        m = new()
        m.load_state_dict(dense, assign=assign)
        made.append(check(m))
    m = Fp8BlockLinear(K, N, transposed=True, device="meta").to_empty(device="cpu")
    check(m).load_state_dict(made[0].state_dict())
    buf = io.BytesIO()
    torch.save(m.state_dict(), buf)
    buf.seek(0)
    n = new()
    n.load_state_dict(torch.load(buf, weights_only=True), assign=True)
    made += [m, n, copy.deepcopy(m), copy.deepcopy(m).half(), torch.nn.Sequential(copy.deepcopy(m)).to(torch.float32)[0]]
    for m in made:
        check(m)
        for t, k in ((m.w_q, "w_q"), (m.w_q_t, "w_q_t")):
            assert torch.equal(t.contiguous().view(torch.uint8), dense[k].view(torch.uint8))
    check(copy.deepcopy(made[0]).to("meta"))


@pytest.mark.parametrize("scaling", [
    {"type": "linear", "factor": 2.0, "attention_factor": 1.2}, {"type": "ntk", "factor": 2.0, "beta_fast": 16.0},
    {"type": "ntk", "factor": 2.0, "beta_slow": 2.0}, {"type": "none", "factor": 2.0},
    {"type": "none", "attention_factor": 1.0}])
def test_rotary_table_refuses_entries_of_another_type(scaling):
    """They were taken and ignored."""
    with pytest.raises(ValueError, match="has no"):
        rotary_table(torch.arange(4), 8, scaling=scaling)


@pytest.mark.parametrize("scaling", [
    {"type": "linear", "factor": 2.0, "original_length": 100}, {"type": "ntk", "factor": 2.0, "original_length": 100},
    {"type": "none"}, {"type": "none", "factor": 1.0, "original_length": 100}, {},
    {"type": "yarn", "factor": 2.0, "original_length": 100, "beta_fast": 16.0, "beta_slow": 2.0, "attention_factor": 1.0}])
def test_rotary_table_takes_its_type_s_entries(scaling):
    with pytest.raises(ValueError, match="CUDA"):  # as far as a tensor on the host goes
        rotary_table(torch.arange(4), 8, scaling=scaling)
