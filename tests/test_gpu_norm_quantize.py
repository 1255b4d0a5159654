"""add_rms_norm_quantize against the formula in 64 bits: types, sizes, groups, strides, what is not finite, what stays as it was."""
import pytest
import torch

from owoinfer_b200 import ops

pytestmark = pytest.mark.gpu

# fp32 steps on the way to a scale, in roundings of 2^-24: the sum of squares is a chain of at most 32 fma, 5 shuffles and 32 warps' sums (69, of which
# the root takes half), the hardware's reciprocal root 2, sum, weight, factor and division one each.
STEP = 2.0 ** -24
SCALE_TOL = 48 * STEP
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
bf16, f16, f32 = torch.bfloat16, torch.float16, torch.float32
int8, e4m3 = torch.int8, torch.float8_e4m3fn


def make(tokens, dim, x_type, r_type, w_type, seed=0, stride=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    def rows(to):
        return torch.randn((tokens, dim + stride), generator=g, device="cuda").to(to)[:, :dim]
    x = rows(x_type)
    r = None if r_type is None else (rows(f32) * 3).to(r_type) if not stride else rows(r_type)
    w = None if w_type is None else (1 + 0.3 * torch.randn(dim, generator=g, device="cuda")).to(w_type)
    return x, r, w


def exact(x, r, w, eps, group, codes):
    s = x.double() if r is None else x.double() + r.double()
    y = s / (s.square().mean(-1, keepdim=True) + eps).sqrt()
    y = y if w is None else y * w.double()
    by = y.view(len(y), -1, group or y.shape[1])
    return s, y, (by.abs().amax(-1) / LARGEST[codes]).clamp(min=1e-30)


def check(x, r, w, codes, group, eps, q, scale, stream, norm, type_of_stream):
    s, y, want = exact(x, r, w, eps, group, codes)
    if stream is not None:
        half = torch.finfo(type_of_stream).eps / 2
        assert ((stream.double() - s).abs() <= s.abs() * (half + STEP) + 2.0 ** -133).all()
    scale = scale.double().view(want.shape)
    assert ((scale - want).abs() <= want * SCALE_TOL).all()
    each = want.repeat_interleave(group or y.shape[1], 1)
    at, got = y / each, q.double()
    wide = at.abs() * 2 * SCALE_TOL  # what the roundings ahead of the last one move
    half = 0.5 if codes == int8 else (at.abs() * 2.0 ** -4).clamp(min=2.0 ** -10)
    assert ((got - at).abs() <= half + wide).all()
    if norm is not None:
        assert ((norm.double() - y).abs() <= y.abs() * (torch.finfo(norm.dtype).eps / 2 + SCALE_TOL) + 2.0 ** -24).all()


@pytest.mark.parametrize("codes", [int8, e4m3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("tokens,dim,x_type,r_type,w_type,group,norm_type,stride", [
    (1, 8, bf16, None, None, 0, None, 0), (3, 16, bf16, bf16, bf16, 0, bf16, 0), (1, 2048, bf16, f32, bf16, 0, None, 0), (130, 272, f16, f32, f16, 0, f16, 8),
    (700, 512, bf16, bf16, f32, 128, None, 16), (2, 768, f32, f32, f32, 256, bf16, 4), (5, 32768, bf16, f32, bf16, 0, bf16, 0), (301, 32768, f32, f32, None, 64, f16, 0),
    (1000, 4096, bf16, f32, bf16, 0, bf16, 0), (999, 8200, f16, f16, f16, 0, None, 8), (400, 5120, bf16, bf16, bf16, 32, None, 0), (1025, 24, bf16, f32, None, 0, bf16, 0),
    (600, 320, f32, None, bf16, 0, f16, 0), (299, 12288, bf16, bf16, bf16, 128, bf16, 0), (297, 96, f16, f32, f32, 32, None, 8), (64, 16384, f32, f32, f32, 0, None, 0),
])
def test_against_the_formula(tokens, dim, x_type, r_type, w_type, group, norm_type, stride, codes):
    x, r, w = make(tokens, dim, x_type, r_type, w_type, seed=tokens + dim, stride=stride)
    norm = None if norm_type is None else torch.empty(tokens, dim, dtype=norm_type, device="cuda")
    out = None if r is None else torch.empty_like(r)
    before = None if r is None else r.clone()
    q, scale = ops.add_rms_norm_quantize(x, w, r, eps=1e-5, dtype=codes, group=group, residual_out=out, norm_out=norm)
    assert q.dtype == codes and q.shape == x.shape and scale.shape == ((tokens, dim // group) if group else (tokens,))
    check(x, r, w, codes, group, 1e-5, q, scale, out, norm, r_type)
    assert r is None or torch.equal(r, before)


def test_in_place_and_into_what_is_read():
    x, r, w = make(300, 1024, bf16, bf16, bf16, seed=5)
    want_stream, want_norm = torch.empty_like(r), torch.empty_like(x)
    want = ops.add_rms_norm_quantize(x, w, r, residual_out=want_stream, norm_out=want_norm)
    stream = r.clone()
    got = ops.add_rms_norm_quantize(x, w, stream)
    assert torch.equal(stream, want_stream) and all(torch.equal(a, b) for a, b in zip(got, want))
    over = x.clone()  # the sum into x
    got = ops.add_rms_norm_quantize(over, w, r, residual_out=over)
    assert torch.equal(over, want_stream) and all(torch.equal(a, b) for a, b in zip(got, want))
    over = x.clone()  # the norm into x
    got = ops.add_rms_norm_quantize(over, w, r.clone(), norm_out=over)
    assert torch.equal(over, want_norm) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_rows_of_wider_matrices_leave_the_rest_alone():
    tokens, dim = 77, 400
    x, r, w = make(tokens, dim, bf16, f32, bf16, seed=9, stride=16)
    q_all, y_all, s_all = (torch.full((tokens + 2, dim + 32), v, dtype=t, device="cuda") for v, t in ((77, int8), (7.0, bf16), (5.0, f32)))
    scale_all = torch.full((tokens + 2,), 3.0, device="cuda")
    q, y, s = (t[1:-1, 16:16 + dim] for t in (q_all, y_all, s_all))
    ops.add_rms_norm_quantize(x, w, r, residual_out=s, norm_out=y, q=q, scale=scale_all[1:-1])
    check(x, r, w, int8, 0, 1e-6, q, scale_all[1:-1], s, y, f32)
    for t, v in ((q_all, 77), (y_all, 7.0), (s_all, 5.0)):
        t = t.clone()
        t[1:-1, 16:16 + dim] = v
        assert (t == v).all()
    assert scale_all[0] == 3.0 and scale_all[-1] == 3.0


@pytest.mark.parametrize("group", [0, 64])
@pytest.mark.parametrize("codes", [int8, e4m3], ids=["int8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 4096])
def test_rows_that_are_not_finite_zero_or_extreme(dim, codes, group):
    x = torch.ones(8, dim, device="cuda") * torch.linspace(-1, 1, dim, device="cuda")
    x[1, 3], x[2, 5], x[3] = float("nan"), float("inf"), 0.0
    x[4] *= 2.0 ** 70                                   # squares past fp32
    x[5] *= 2.0 ** (60 - (dim.bit_length() + 1) // 2)   # just inside
    x[6] *= 1e-20                                       # eps is all of the mean
    q, scale = ops.add_rms_norm_quantize(x, eps=1e-6, dtype=codes, group=group, norm_out=(y := torch.empty(8, dim, dtype=bf16, device="cuda")))
    scale = scale.view(8, -1)
    for row in (1, 2, 4):
        assert scale[row].isnan().all() and y[row].isnan().all()
        assert (q[row] == 0).all() if codes == int8 else q[row].float().isnan().all()
    assert (scale[3] == torch.tensor(1e-30, device="cuda")).all() and (q[3].float() == 0).all() and (y[3] == 0).all()
    fine = torch.tensor([0, 5, 6, 7], device="cuda")
    check(x[fine], None, None, codes, group, 1e-6, q[fine], scale[fine].view(-1) if not group else scale[fine], None, y[fine], None)


@pytest.mark.parametrize("group", [0, 32])
def test_zeros_without_an_eps(group):
    x = torch.ones(3, 64, device="cuda", dtype=bf16)
    x[1] = 0
    q, scale = ops.add_rms_norm_quantize(x, eps=0.0, group=group)
    assert scale[1].isnan().all() and (q[1] == 0).all() and (q[::2] == 127).all() and ((scale[::2] * 127 - 1).abs() < 1e-6).all()


def test_no_tokens_and_a_captured_call_on_another_stream():
    q, scale = ops.add_rms_norm_quantize(torch.empty(0, 64, dtype=bf16, device="cuda"), group=32)
    assert q.shape == (0, 64) and scale.shape == (0, 2)
    x, r, w = make(9, 2048, bf16, f32, bf16, seed=3)
    out = torch.empty_like(r)
    want = ops.add_rms_norm_quantize(x, w, r, residual_out=out)
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        got = ops.add_rms_norm_quantize(x, w, r, residual_out=out)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
