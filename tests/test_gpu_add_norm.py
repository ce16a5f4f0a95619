"""b200::add_rms_norm and add_rms_norm_quant against the formula in 64 bits.

Bounds.  sum: bit-equal to the rounded addition.  out: the fp32 sum of
squares, square root and products err by less than 2e-5 relative (chains of
at most 64 fp32 additions, 64 * 2^-24 / 2, plus a few single roundings), then
half a step of the output type for each rounding (one; two with
ROUND_NORMED).  e4m3: half a step, 2^-4 relative or 2^-10 of a scale below
the smallest normal number."""
import pytest
import torch

import serving_reference as ref
from compiler import runtime
from compiler.runtime import cabi

pytestmark = pytest.mark.gpu
runtime.load()
FP32 = 2e-5
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def make(rows, cols, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + rows * 7 + cols)
    x = torch.randn(rows, cols, device="cuda", generator=g).to(dtype)
    r = (3 * torch.randn(rows, cols, device="cuda", generator=g)).to(dtype)
    w = (1 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(dtype)
    return x, r, w


def check(out, total, x, r, w, eps, flags=0):
    want_sum, y = ref.add_rms_norm(x, r, w, eps, plus_one=bool(flags & 8))
    assert torch.equal(total, want_sum)
    h = ref.HALF_STEP[x.dtype]
    roundings = (2 if flags & 1 else 1) * h * 1.01  # the product of two roundings is below 1.01 of their sum
    tiny = 2.0**-24 if x.dtype == torch.float16 else 0.0  # fp16 subnormals step by 2^-24
    assert ((out.double() - y).abs() <= y.abs() * (roundings + FP32) + tiny).all()


SHAPES = [(1, 8), (1, 1), (3, 7), (1, 2048), (5, 4096), (17, 100), (33, 520), (4, 1000), (9, 1024), (2, 4104),
          (3, 5001), (2, 8192), (2, 16384), (1, 32768), (1, 40000), (300, 768), (2, 12289)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_against_the_formula(rows, cols, dtype):
    x, r, w = make(rows, cols, dtype)
    out, total = torch.ops.b200.add_rms_norm(x, r, w, 1e-5)
    check(out, total, x, r, w, 1e-5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 2, 13])
@pytest.mark.parametrize("cols", [1, 2, 63, 126, 127, 129, 255, 510, 511, 513, 1022, 1023, 1025, 2047, 2049, 4095, 4097,
                                  6143, 6145, 12289])
def test_odd_widths(cols, rows, dtype):
    """Rows shared out among 32 to 512 threads, several in a CTA and not a
    multiple of them, either half of a word first."""
    x, r, w = make(rows, cols, dtype)
    out, total = torch.ops.b200.add_rms_norm(x, r, w, 1e-5)
    check(out, total, x, r, w, 1e-5)
    q, scale, total = torch.ops.b200.add_rms_norm_quant(x, r, w, 1e-5)
    check_quant(q, scale, total, x, r, w, 0)


@pytest.mark.parametrize("flags", [1, 8, 9])
@pytest.mark.parametrize("cols", [1024, 99])
def test_flags(cols, flags):
    x, r, w = make(6, cols, torch.bfloat16)
    out, total = torch.ops.b200.add_rms_norm(x, r, w, 1e-5, flags)
    check(out, total, x, r, w, 1e-5, flags)


@pytest.mark.parametrize("cols", [512, 33])
def test_without_weight_and_with_a_fp32_weight(cols):
    x, r, w = make(6, cols, torch.float16)
    for weight in (None, w.float()):
        out, total = torch.ops.b200.add_rms_norm(x, r, weight, 1e-6)
        check(out, total, x, r, weight, 1e-6)


def check_quant(q, scale, total, x, r, w, group):
    want_sum, y = ref.add_rms_norm(x, r, w, 1e-5)
    assert torch.equal(total, want_sum)
    cols = x.shape[1]
    width = group or cols
    top = y.abs().unflatten(1, (-1, width)).amax(-1).clamp_min(1e-12)
    assert ((scale.double() - top / 448).abs() <= top / 448 * FP32).all()
    s = scale.double().repeat_interleave(width, 1)
    err = (q.double() * s - y).abs()
    assert (err <= y.abs() * (2.0**-4 + 1e-4) + s * 2.0**-10 * (1 + 1e-4)).all()
    assert q.float().abs().unflatten(1, (-1, width)).amax(-1).eq(448).all()  # the largest is the type's largest


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,group", [(1, 128, 128), (5, 2048, 0), (7, 4096, 128), (3, 77, 0), (2, 8192, 128),
                                             (2, 1152, 128), (1, 5001, 0), (2, 40064, 128), (2, 40000, 0), (130, 256, 0)])
def test_quant(rows, cols, group, dtype):
    x, r, w = make(rows, cols, dtype)
    q, scale, total = torch.ops.b200.add_rms_norm_quant(x, r, w, 1e-5, group)
    check_quant(q, scale, total, x, r, w, group)


@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("offset", [0, 1])
def test_quant_of_unaligned_rows(group, offset):
    x, r, w = make(5, 512 + 8, torch.bfloat16)
    x, r, w = x[:, offset:offset + 512], r[:, 8 - offset:520 - offset], w[offset:offset + 512]
    q, scale, total = torch.ops.b200.add_rms_norm_quant(x, r, w, 1e-5, group)
    check_quant(q, scale, total, x, r, w, group)


def test_rows_of_zeros_infinities_and_nan():
    x, r, w = make(4, 1024, torch.bfloat16)
    x[0], r[0] = 0, 0
    x[1, 5] = float("inf")
    x[2, 700] = float("nan")
    for cols in (1024, 1023):  # the vector and the element kernel
        a, b, c = x[:, :cols].contiguous(), r[:, :cols].contiguous(), w[:cols].contiguous()
        q, scale, total = torch.ops.b200.add_rms_norm_quant(a, b, c, 1e-5)
        assert q[0].float().abs().max() == 0 and scale[0].item() == pytest.approx(1e-12 / 448, rel=1e-5)
        assert scale[1:3].isnan().all() and q.float()[2].isnan().all() and q.float()[1, 5].isnan()
        assert scale[3].isfinite().all() and q.float()[3].isfinite().all()
        out, _ = torch.ops.b200.add_rms_norm(a, b, c, 1e-5)
        assert out[0].abs().max() == 0 and out[2].isnan().all() and out[3].isfinite().all()


def test_strided_and_three_dimensional_rows():
    x, r, w = make(12, 1024, torch.bfloat16)
    for view in (lambda t: t.view(3, 4, 1024), lambda t: t[::2], lambda t: t[:, 100:356],
                 lambda t: t.view(3, 4, 1024).transpose(0, 1), lambda t: t[:, ::2], lambda t: t[0]):
        a, b = view(x), view(r)
        weight = w[:a.shape[-1]]
        out, total = torch.ops.b200.add_rms_norm(a, b, weight, 1e-5)
        assert out.shape == a.shape and total.is_contiguous()
        check(out.reshape(-1, a.shape[-1]), total.reshape(-1, a.shape[-1]), a.reshape(-1, a.shape[-1]),
              b.reshape(-1, a.shape[-1]), weight, 1e-5)


def test_an_expanded_residual_and_empty_rows():
    x, r, w = make(6, 256, torch.float16)
    out, total = torch.ops.b200.add_rms_norm(x, r[:1].expand(6, 256), w, 1e-5)
    check(out, total, x, r[:1].expand(6, 256), w, 1e-5)
    out, total = torch.ops.b200.add_rms_norm(x[:0], r[:0], w, 1e-5)
    assert out.shape == total.shape == (0, 256)


def test_equals_the_addition_followed_by_rms_norm():
    """The fused result is the library's norm of the rounded sum, up to the
    order of the row sum (one step of the output type at most)."""
    x, r, w = make(64, 2048, torch.bfloat16)
    out, total = torch.ops.b200.add_rms_norm(x, r, w, 1e-5, 1)
    two = torch.ops.b200.rms_norm(x + r, w, 1e-5, 1, torch.bfloat16)
    assert torch.equal(total, x + r)
    assert ((out.float() - two.float()).abs() <= two.float().abs() * 2.0**-7).all()
    assert (out == two).float().mean() > 0.999


def test_refusals():
    x, r, w = make(4, 256, torch.bfloat16)
    for bad in (lambda: torch.ops.b200.add_rms_norm(x, r[:3], w, 1e-5),
                lambda: torch.ops.b200.add_rms_norm(x, r.float(), w, 1e-5),
                lambda: torch.ops.b200.add_rms_norm(x, r, w[:8], 1e-5),
                lambda: torch.ops.b200.add_rms_norm(x, r, w.cpu(), 1e-5),
                lambda: torch.ops.b200.add_rms_norm(x.double(), r.double(), w, 1e-5),
                lambda: torch.ops.b200.add_rms_norm(x, r, w, 1e-5, 2),
                lambda: torch.ops.b200.add_rms_norm_quant(x, r, w, 1e-5, 64),
                lambda: torch.ops.b200.add_rms_norm_quant(x[:, :200], r[:, :200], w[:200], 1e-5, 128),
                lambda: torch.ops.b200.add_rms_norm(x.clone().requires_grad_(), r, w, 1e-5)):
        with pytest.raises(RuntimeError):
            bad()


def test_c_abi_and_another_stream():
    x, r, w = make(40, 4096, torch.bfloat16)
    total, out = torch.empty_like(x), torch.empty_like(x, dtype=torch.float8_e4m3fn)
    scale = torch.empty(40, 32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cabi.add_rms_norm(x, r, w, 1e-5, total, out, scale, 128)
    side.synchronize()
    check_quant(out, scale, total, x, r, w, 128)


def test_dims_of_one_element_have_no_say_in_flattening():
    """[4, 1, 3, cols] cut from four rows of each of four blocks: the size-one
    dim's stride looks like a row stride and is none."""
    x, r, w = make(16, 256, torch.bfloat16)
    a, b = x.view(4, 1, 4, 256)[:, :, :3], r.view(4, 1, 4, 256)[:, :, :3]
    out, total = torch.ops.b200.add_rms_norm(a, b, w, 1e-5)
    check(out.reshape(12, 256), total.reshape(12, 256), a.reshape(12, 256), b.reshape(12, 256), w, 1e-5)
    a, b = x.view(16, 1, 256)[::2], r.view(16, 1, 256)[1::2]
    out, total = torch.ops.b200.add_rms_norm(a, b, w, 1e-5)
    check(out.reshape(8, 256), total.reshape(8, 256), a.reshape(8, 256), b.reshape(8, 256), w, 1e-5)
