"""The training operators against their definitions in 64 bits.

Tolerances.  u is the unit roundoff of the stored type (2^-24, 2^-11, 2^-8).
A result is one rounding of an fp32 value (u / sqrt(3) of its norm at most for
values spread over a binade, u at worst), and in 16-bit types the matrix
products take their operands (probabilities, score gradients) in that type,
one more rounding: 2 u of the norm.  fp32 results: scores of magnitude up to
about 8 carry an error of some ulps of 8, which the exponential turns into a
relative error: 1e-5 of the norm.  Values that are sums with cancellation
(one token: the score gradient is zero) get an absolute term of 16 fp32 ulps
of the terms, whose magnitude is D (a product of two D-vectors), times the root
of how many pairs are summed for the bias tables.
"""
import math

import pytest
import torch

from . import train_ops_reference as ref

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = list(U)


def rel(dtype):
    return max(1e-5, 2 * U[dtype])


def close(got, want, rtol, atol=0.0):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    off, norm = (got - want).norm().item(), want.norm().item()
    assert off <= rtol * norm + atol * math.sqrt(max(1, want.numel())), (off, norm, rtol, atol)


def attention_inputs(b, n, nq, h, d, dtype, seed=0, clip=8, clip_z=2, holes=False, table_dtype=torch.float32,
                     spread=6):
    g = torch.Generator("cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda")

    qkv = randn(b, n, 3, h, d).to(dtype)
    mask = torch.rand(b, n, generator=g, device="cuda") < 0.7
    if not holes:
        mask = torch.arange(n, device="cuda")[None] < mask.sum(1, keepdim=True).clamp_min(1)
    mask[:, 0] = True
    at = [torch.randint(-spread, spread + 1, (b, n), generator=g, device="cuda", dtype=torch.int32) for _ in range(3)]
    tables = [(0.5 * randn(2 * c + 1, h)).to(table_dtype) for c in (clip, clip, clip_z)]
    dout = randn(b, nq, h, d).to(dtype)
    return qkv, [*at, mask], tables, dout


def check_attention(q, k, v, where, tables, dout, scale=None):
    from hive_neuralnet_b200 import train_ops as ops
    dtype, (b, nq, h, d), n = q.dtype, q.shape, k.shape[1]
    out, saved = ops.relative_attention_forward(q, k, v, *where, *tables, scale=scale, save=True)
    alone, none = ops.relative_attention_forward(q, k, v, *where, *tables, scale=scale)
    assert none is None and torch.equal(out, alone)
    got = [out, *ops.relative_attention_backward(dout, q, k, v, *where, *tables, saved, scale=scale)]
    again = ops.relative_attention_backward(dout, q, k, v, *where, *tables, saved, scale=scale)
    assert all(torch.equal(x, y) for x, y in zip(got[1:], again))
    want = ref.attention_grads(dout, q, k, v, *where, *tables, scale=scale)
    for i, (x, y) in enumerate(zip(got, want)):
        if i < 4:
            close(x, y, rel(dtype), 16 * U[torch.float32] * d)
        else:
            assert x.dtype == tables[i - 4].dtype
            close(x, y, rel(x.dtype), 16 * U[torch.float32] * d * math.sqrt(b * nq * n))
    dead = ~where[3].bool()
    if b and n:
        assert not out[dead[:, :nq]].any() and not got[1][dead[:, :nq]].any()
        assert not got[2][dead].any() and not got[3][dead].any()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,n,nq,h,d", [
    (1, 1, 1, 1, 8), (3, 2, 2, 1, 1), (5, 7, 7, 3, 4), (2, 8, 8, 8, 8), (3, 15, 15, 2, 16), (3, 16, 16, 8, 8),
    (2, 17, 17, 5, 12), (9, 29, 29, 8, 8), (4, 29, 29, 8, 16), (3, 29, 1, 8, 8), (2, 31, 5, 1, 33), (2, 32, 32, 2, 64),
    (2, 33, 33, 2, 8), (2, 33, 1, 3, 24), (1, 64, 64, 2, 32), (2, 65, 65, 2, 64), (2, 70, 19, 2, 48), (1, 127, 127, 1, 7),
    (1, 130, 130, 2, 16), (1, 257, 257, 2, 64), (1, 300, 1, 2, 64), (1, 513, 200, 1, 40)])
def test_attention(b, n, nq, h, d, dtype):
    qkv, where, tables, dout = attention_inputs(b, n, nq, h, d, dtype, seed=n + d, holes=n % 2 == 0)
    q, k, v = qkv.unbind(2)
    check_attention(q[:, :nq], k, v, where, tables, dout)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_many_positions(dtype):
    """More work than one wave of blocks: the loops over positions, the partial bias sums."""
    qkv, where, tables, dout = attention_inputs(3001, 29, 29, 8, 8, dtype, seed=5)
    check_attention(*qkv.unbind(2), where, tables, dout)


@pytest.mark.parametrize("clip,clip_z", [(0, 0), (1, 2), (16, 4), (3, 0)])
@pytest.mark.parametrize("n", [29, 90])
def test_attention_clips(clip, clip_z, n):
    qkv, where, tables, dout = attention_inputs(3, n, n, 3, 8, torch.float32, clip=clip, clip_z=clip_z, spread=20)
    check_attention(*qkv.unbind(2), where, tables, dout, scale=0.3)


@pytest.mark.parametrize("n", [29, 100])
def test_attention_far_coordinates(n):
    """Coordinates over the whole int32 range are clamped; int64 ones too."""
    qkv, where, tables, dout = attention_inputs(2, n, n, 2, 8, torch.float32)
    for t in where[:3]:
        t[:, ::3] = 2 ** 31 - 1
        t[:, 1::3] = -2 ** 31
    got = check_attention(*qkv.unbind(2), where, tables, dout)
    far = [t.long() * 1000 for t in where[:3]]
    near = [t.clamp(-2 ** 19, 2 ** 19) for t in where[:3]]
    from hive_neuralnet_b200 import train_ops as ops
    big, _ = ops.relative_attention_forward(*qkv.unbind(2), *[f.clamp(-2 ** 40, 2 ** 40) for f in far], where[3], *tables)
    want, _ = ops.relative_attention_forward(*qkv.unbind(2), *[f.clamp(-2 ** 19, 2 ** 19).int() for f in far], where[3],
                                             *tables)
    assert torch.equal(big, want)
    same, _ = ops.relative_attention_forward(*qkv.unbind(2), *near, where[3], *tables)
    assert torch.equal(same, got[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,fill", [(29, float("nan")), (29, float("inf")), (29, "lowest"), (90, float("nan")),
                                    (90, "lowest")])
def test_attention_masked_places_hold_anything(n, fill, dtype):
    qkv, where, tables, dout = attention_inputs(4, n, n, 3, 16, dtype, holes=True)
    where[3][1] = False  # a position with no token
    where[3][2] = False
    where[3][2, n - 1] = True  # one token, the last
    clean = check_attention(*qkv.unbind(2), where, tables, dout)
    value = torch.finfo(dtype).min if fill == "lowest" else fill
    bad, bad_dout = qkv.clone(), dout.clone()
    bad[~where[3]] = value
    bad_dout[~where[3]] = value
    got = check_attention(*bad.unbind(2), where, tables, bad_dout)
    assert all(torch.equal(x, y) for x, y in zip(got, clean))
    bad_at = [torch.where(where[3], t, torch.full_like(t, 2 ** 31 - 1)) for t in where[:3]]
    got = check_attention(*bad.unbind(2), [*bad_at, where[3]], tables, bad_dout)
    assert all(torch.equal(x, y) for x, y in zip(got, clean))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [29, 70])
def test_attention_layouts(n, dtype):
    """Head-major operands, rows and bases off 16-byte boundaries, tokens shared by the batch, uint8 masks."""
    from hive_neuralnet_b200 import train_ops as ops
    b, h, d = 3, 4, 8
    qkv, where, tables, dout = attention_inputs(b, n, n, h, d, dtype)
    where = [t[:1].expand(b, n) for t in where]
    want = check_attention(*qkv.unbind(2), where, tables, dout)
    head_major = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (*qkv.unbind(2), dout)]
    wide = torch.zeros(b, n, h, d + 3, dtype=dtype, device="cuda")
    wide[..., 1:d + 1] = qkv[:, :, 0]
    odd = torch.zeros(b * n * h * d + 1, dtype=dtype, device="cuda")[1:].view(b, n, h, d)
    odd.copy_(qkv[:, :, 2])
    gaps = torch.zeros(b, n, h, 2 * d, dtype=dtype, device="cuda")[..., ::2]
    gaps.copy_(qkv[:, :, 1])
    u8 = [*where[:3], where[3].to(torch.uint8) * 255]
    for q, k, v, do in ((*head_major,), (wide[..., 1:d + 1], gaps, odd, dout)):
        out, saved = ops.relative_attention_forward(q, k, v, *u8, *tables, save=True)
        got = [out, *ops.relative_attention_backward(do, q, k, v, *u8, *tables, saved)]
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    # one set of keys for the whole batch (batch stride 0)
    q, k, v = qkv.unbind(2)
    check_attention(q, k[:1].expand(b, n, h, d), v[:1].expand(b, n, h, d), where, tables, dout)


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_attention_tables_in_the_type_of_q(dtype):
    for n in (29, 70):
        qkv, where, tables, dout = attention_inputs(3, n, n, 2, 8, dtype, table_dtype=dtype)
        check_attention(*qkv.unbind(2), where, tables, dout)


@pytest.mark.parametrize("n", [29, 80])
def test_attention_strong_scores(n):
    """Scores far apart (one key takes all) and a large common offset."""
    qkv, where, tables, dout = attention_inputs(3, n, n, 2, 8, torch.float32)
    q, k, v = qkv.unbind(2)
    from hive_neuralnet_b200 import train_ops as ops
    tables = [t + 200.0 for t in tables]
    out, saved = ops.relative_attention_forward(40 * q, k, v, *where, *tables, save=True)
    got = [out, *ops.relative_attention_backward(dout, 40 * q, k, v, *where, *tables, saved)]
    want = ref.attention_grads(dout, 40 * q, k, v, *where, *tables)
    # scores of 700 have ulps of 2^-14: 40 times coarser probabilities than the scores of 8 above
    for x, y in zip(got[:4], want[:4]):
        close(x, y, 1e-3)


def test_attention_empty():
    from hive_neuralnet_b200 import train_ops as ops
    for b, n, nq in ((0, 29, 29), (2, 0, 0), (2, 5, 0)):
        qkv, where, tables, dout = attention_inputs(b, max(n, 1), nq, 2, 8, torch.float32)
        q, k, v = qkv[:, :n].unbind(2)
        where = [t[:, :n] for t in where]
        out, saved = ops.relative_attention_forward(q[:, :nq], k, v, *where, *tables, save=True)
        grads = ops.relative_attention_backward(dout[:, :nq], q[:, :nq], k, v, *where, *tables, saved)
        assert out.shape == (b, nq, 2, 8)
        assert not any(g.any() for g in grads)


def test_attention_no_queries_of_many_tokens():
    qkv, where, tables, dout = attention_inputs(2, 40, 0, 3, 8, torch.float32)
    got = check_attention(qkv[:, :0, 0], qkv[:, :, 1], qkv[:, :, 2], where, tables, dout)
    assert not any(t.any() for t in got[2:])


@pytest.mark.parametrize("n", [29, 70])
def test_attention_tables_written_just_before(n):
    """Each pass follows at once on the kernels that write its bias tables and operands."""
    from hive_neuralnet_b200 import train_ops as ops
    qkv, where, tables, dout = attention_inputs(40, n, n, 8, 16, torch.bfloat16)
    out, saved = ops.relative_attention_forward(*qkv.unbind(2), *where, *tables, save=True)
    want = [out, *ops.relative_attention_backward(dout, *qkv.unbind(2), *where, *tables, saved)]
    late, spare = [t.clone() for t in tables], torch.zeros(50_000_000, device="cuda")
    for _ in range(3):
        for t in late:
            t.zero_()
        torch.cuda.synchronize()
        spare.add_(1)
        for t, value in zip(late, tables):
            t.copy_(value)
        out, saved = ops.relative_attention_forward(*qkv.unbind(2), *where, *late, save=True)
        for t in late:
            t.zero_()
        spare.add_(1)
        for t, value in zip(late, tables):
            t.copy_(value)
        got = [out, *ops.relative_attention_backward(dout, *qkv.unbind(2), *where, *late, saved)]
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_types_in_turn_in_a_new_process():
    """A kernel's first launch in a process, of one type after another at the same shape."""
    import subprocess
    import sys
    code = """
import torch
from hive_neuralnet_b200 import train_ops as ops
for n in (29, 70):
    for dtype in (torch.float16, torch.bfloat16, torch.float32, torch.float16):
        qkv = torch.ones(3, n, 3, 8, 64, device='cuda', dtype=dtype)
        at, mask = torch.zeros(3, n, dtype=torch.int32, device='cuda'), torch.ones(3, n, dtype=torch.bool, device='cuda')
        tables = [torch.zeros(17, 8, device='cuda'), torch.zeros(17, 8, device='cuda'), torch.zeros(5, 8, device='cuda')]
        q, k, v = qkv.unbind(2)
        out, saved = ops.relative_attention_forward(q, k, v, at, at, at, mask, *tables, save=True)
        grads = ops.relative_attention_backward(out, q, k, v, at, at, at, mask, *tables, saved)
        assert (out.float() - 1).abs().max().item() < 1e-2 and grads[0].abs().max().item() < 1e-2
        x = qkv.reshape(-1, 64)
        y, s, mean, rstd = ops.layer_norm_forward(x, torch.ones(64, device='cuda'), torch.zeros(64, device='cuda'))
        ops.layer_norm_backward(y, s, torch.ones(64, device='cuda'), mean, rstd)
        torch.cuda.synchronize()
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_attention_offsets_past_32_bits():
    """Batch strides over 2^31 elements."""
    b, n, h, d = 2, 29, 8, 8
    qkv, where, tables, dout = attention_inputs(b, n, n, h, d, torch.float16)
    stride = 2 ** 31 + 64
    big = torch.empty(stride + 3 * n * h * d, dtype=torch.float16, device="cuda")
    far = big.as_strided((b, n, 3, h, d), (stride, 3 * h * d, h * d, d, 1))
    far.copy_(qkv)
    want = check_attention(*qkv.unbind(2), where, tables, dout)
    got = check_attention(*far.unbind(2), where, tables, dout)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("n", [29, 70])
def test_attention_by_differences(n):
    """Directional differences of sum(out * dout) in each input, steps of 2^-8 in fp32:
    truncation (step^2 times third derivatives of order 10) 2e-4 of the gradient's
    size, rounding of the sum 2^-24 / 2^-8 of its terms."""
    from hive_neuralnet_b200 import train_ops as ops
    qkv, where, tables, dout = attention_inputs(2, n, n, 2, 8, torch.float32)
    args = [*qkv.unbind(2), *tables]

    def value(a):
        out, _ = ops.relative_attention_forward(*a[:3], *where, *a[3:])
        return (out.double() * dout.double()).sum().item()

    _, saved = ops.relative_attention_forward(*args[:3], *where, *args[3:], save=True)
    grads = ops.relative_attention_backward(dout, *args[:3], *where, *args[3:], saved)
    g = torch.Generator("cuda").manual_seed(1)
    step = 2.0 ** -8
    for i, grad in enumerate(grads):
        way = torch.randn(args[i].shape, generator=g, device="cuda").sign()
        plus = value([a + step * way if j == i else a for j, a in enumerate(args)])
        minus = value([a - step * way if j == i else a for j, a in enumerate(args)])
        want = (grad.double() * way.double()).sum().item()
        size = grad.double().norm().item() + dout.norm().item() * 2.0 ** -16 / step
        assert abs((plus - minus) / (2 * step) - want) <= 2e-3 * size, i


@pytest.mark.parametrize("n", [29, 70])
def test_attention_autograd_and_the_module(n):
    """The autograd forms against the network's own attention module on the valid tokens."""
    from hive_neuralnet_b200 import train_ops as ops
    from hive_neuralnet_b200.hybrid import RelativeSelfAttention
    torch.manual_seed(3)
    m = RelativeSelfAttention(64, 8, 8, 2).cuda()
    _, where, _, _ = attention_inputs(5, n, n, 8, 8, torch.float32)
    live = where[3][:, :, None]
    x = torch.randn(5, n, 64, device="cuda", requires_grad=True)
    dy = torch.randn(5, n, 64, device="cuda") * live
    tables = [t.weight for t in (m.dq_bias, m.dr_bias, m.dz_bias)]
    names = [x, *m.parameters()]
    want_y = m(x, *[t.long() for t in where[:3]], where[3])
    want = torch.autograd.grad(want_y, names, dy)
    for packed in (True, False):
        qkv = m.qkv(x).view(5, n, 3, 8, 8)
        o = (ops.relative_attention_packed(qkv, *where, *tables) if packed
             else ops.relative_attention(*qkv.unbind(2), *where, *tables))
        y = m.out_proj(o.flatten(2))
        close(y * live, want_y * live, 1e-5)
        for g, w in zip(torch.autograd.grad(y, names, dy), want):
            close(g, w, 2e-5, 1e-6)  # two fp32 paths, each 1e-5


@pytest.mark.parametrize("n", [29, 70])
def test_attention_on_another_stream(n):
    from hive_neuralnet_b200 import train_ops as ops
    qkv, where, tables, dout = attention_inputs(600, n, n, 8, 8, torch.float16)
    _, saved = ops.relative_attention_forward(*qkv.unbind(2), *where, *tables, save=True)
    want = ops.relative_attention_backward(dout, *qkv.unbind(2), *where, *tables, saved)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = qkv.clone()
        torch.cuda._sleep(20_000_000)
        late.mul_(1)
        out, saved = ops.relative_attention_forward(*late.unbind(2), *where, *tables, save=True)
        got = ops.relative_attention_backward(dout, *late.unbind(2), *where, *tables, saved)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [
    (1, 1), (5, 1), (1, 64), (29, 64), (1000, 64), (33, 8), (7, 2), (50, 3), (100, 31), (64, 96), (300, 128), (17, 200),
    (40, 256), (13, 257), (9, 512), (5, 513), (6, 1000), (21, 1024), (3, 1025), (10, 2047), (4, 2048), (3, 4097),
    (5, 8192), (2, 8191), (70001, 64), (5000, 65), (0, 64)])
def test_norm(rows, width, dtype):
    from hive_neuralnet_b200 import train_ops as ops
    g = torch.Generator("cuda").manual_seed(rows + width)

    def randn(*s):
        return torch.randn(*s, generator=g, device="cuda")

    for residual in (False, True):
        for wt in {torch.float32, dtype}:
            x = (randn(rows, width) * 2 + 1).to(dtype)
            r = randn(rows, width).to(dtype) if residual else None
            w, b = (1 + 0.3 * randn(width)).to(wt), randn(width).to(wt)
            dy, ds = randn(rows, width).to(dtype), randn(rows, width).to(dtype) if residual else None
            y, s, mean, rstd = ops.layer_norm_forward(x, w, b, 1e-5, residual=r)
            assert torch.equal(s, (x.float() + r.float()).to(dtype) if residual else x)
            grads = ops.layer_norm_backward(dy, s, w, mean, rstd, dsum=ds)
            again = ops.layer_norm_backward(dy, s, w, mean, rstd, dsum=ds)
            assert all(torch.equal(a, c) for a, c in zip(grads, again))
            want = ref.norm(s, w, b, 1e-5, dy, ds)
            # width 1 and 2: the centred values cancel, rstd is up to 1/sqrt(eps) = 316 and dx a
            # difference of terms of size rstd
            scale = 316.0 if width < 8 else 1.0
            for got, exact, t in zip((y, *grads), want, (dtype, dtype, wt, wt)):
                assert got.dtype == t
                close(got, exact, rel(t), 16 * U[torch.float32] * scale * (1 if got.dim() > 1 else math.sqrt(max(rows, 1))))


def test_norm_shifted_rows():
    """Rows whose mean is 1000 times their spread: the variance is that of the centred
    values.  x is exact in fp32; its centred value has an error of some ulps of 1000."""
    from hive_neuralnet_b200 import train_ops as ops
    x = 1000 + torch.randn(100, 96, device="cuda")
    w, b = torch.ones(96, device="cuda"), torch.zeros(96, device="cuda")
    y, *_ = ops.layer_norm_forward(x, w, b)
    close(y, ref.norm(x, w, b, 1e-5, x)[0], 4 * 1000 * U[torch.float32])


def test_norm_layouts_and_autograd():
    """Leading axes, non-contiguous inputs, bases off 16-byte boundaries; torch's layer norm in fp64."""
    from hive_neuralnet_b200 import train_ops as ops
    x = torch.randn(6, 29, 64, device="cuda")
    w, b = torch.randn(64, device="cuda", requires_grad=True), torch.randn(64, device="cuda", requires_grad=True)
    want, _, mean, _ = ops.layer_norm_forward(x, w.detach(), b.detach())
    assert mean.shape == (6, 29)
    turned = x.permute(2, 0, 1).contiguous().permute(1, 2, 0)
    odd = torch.zeros(x.numel() + 1, device="cuda")[1:].view_as(x).copy_(x)
    assert torch.equal(ops.layer_norm_forward(turned, w.detach(), b.detach())[0], want)
    close(ops.layer_norm_forward(odd, w.detach(), b.detach())[0], want, 1e-6)
    x.requires_grad_()
    r = torch.randn(6, 29, 64, device="cuda", requires_grad=True)
    y, s = ops.layer_norm(x, w, b, residual=r)
    dy, ds = torch.randn_like(y), torch.randn_like(y)
    got = torch.autograd.grad((y * dy).sum() + (s * ds).sum(), (x, r, w, b))
    x64, r64, w64, b64 = (t.detach().double().requires_grad_() for t in (x, r, w, b))
    s64 = x64 + r64
    y64 = torch.nn.functional.layer_norm(s64, (64,), w64, b64)
    exact = torch.autograd.grad((y64 * dy).sum() + (s64 * ds).sum(), (x64, r64, w64, b64))
    for g, e in zip(got, exact):
        close(g, e, 1e-5)
    y, s = ops.layer_norm(x, w, b, residual=r)
    assert torch.equal(torch.autograd.grad(s.sum(), r)[0], torch.ones_like(r))  # only the sum used
    close(torch.autograd.grad(ops.layer_norm(x, w, b).square().sum(), x)[0],
          torch.autograd.grad(torch.nn.functional.layer_norm(x64, (64,), w64, b64).square().sum(), x64)[0], 1e-5, 1e-5)


def test_norm_by_differences():
    """As for the attention: steps of 2^-8, third derivatives of order 10."""
    from hive_neuralnet_b200 import train_ops as ops
    g = torch.Generator("cuda").manual_seed(2)
    args = [torch.randn(50, 96, generator=g, device="cuda"), 1 + 0.2 * torch.randn(96, generator=g, device="cuda"),
            torch.randn(96, generator=g, device="cuda")]
    dy = torch.randn(50, 96, generator=g, device="cuda")
    _, s, mean, rstd = ops.layer_norm_forward(*args)
    grads = ops.layer_norm_backward(dy, s, args[1], mean, rstd)
    step = 2.0 ** -8

    def value(a):
        return (ops.layer_norm_forward(*a)[0].double() * dy.double()).sum().item()

    for i, grad in enumerate(grads):
        way = torch.randn(args[i].shape, generator=g, device="cuda").sign()
        diff = value([a + step * way if j == i else a for j, a in enumerate(args)]) \
            - value([a - step * way if j == i else a for j, a in enumerate(args)])
        size = grad.double().norm().item() + dy.norm().item() * 2.0 ** -16 / step
        assert abs(diff / (2 * step) - (grad.double() * way.double()).sum().item()) <= 2e-3 * size, i


def test_norm_offsets_past_32_bits():
    from hive_neuralnet_b200 import train_ops as ops
    rows, width = 1_050_000, 2050  # 2.15e9 values
    x = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda").normal_()
    w, b = torch.ones(width, device="cuda"), torch.zeros(width, device="cuda")
    y, s, mean, rstd = ops.layer_norm_forward(x, w, b)
    dx, dw, db = ops.layer_norm_backward(y, s, w, mean, rstd)
    tail = slice(rows - 50, rows)
    want = ref.norm(x[tail], w, b, 1e-5, y[tail])
    close(y[tail], want[0], rel(x.dtype))
    close(dx[tail], want[1], rel(x.dtype), 2 * U[x.dtype])  # dy = y: the terms cancel, of size one
    close(dw, torch.full_like(dw, float(rows)), 1e-2)


# ---------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------
HYPER = dict(lr=3e-3, betas=(0.9, 0.995), eps=1e-8, weight_decay=0.02)


def parts(flat, params):
    out, o = [], 0
    for p in params:
        out.append(flat[o:o + p.numel()])
        o += -(-p.numel() // 256) * 256
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [255, 256, 257], [0, 3, 0], [5000], [64 * 64, 64, 1, 17, 100_003],
                                   list(range(1, 200)), [300] * 1500])
def test_adamw_32(sizes, dtype):
    from hive_neuralnet_b200 import train_ops as ops
    g = torch.Generator("cuda").manual_seed(len(sizes))
    params = [torch.randn(n, generator=g, device="cuda").to(dtype) for n in sizes]
    m, v = (torch.zeros(ops.state_size(params), device="cuda") for _ in range(2))
    steps = 3 if len(sizes) < 1000 else 1
    for step in range(1, steps + 1):
        grads = [(0.1 * torch.randn(n, generator=g, device="cuda")).to(dtype) for n in sizes]
        before = [(p.clone(), a.clone(), b.clone()) for p, a, b in zip(params, parts(m, params), parts(v, params))]
        ops.adamw_step(params, grads, m, v, step=step, **HYPER)
        want = [ref.adamw(p, gr, a, b, step, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
                for (p, a, b), gr in zip(before, grads)]
        for got, i in ((params, 0), (parts(m, params), 1), (parts(v, params), 2)):
            # a product and a sum each rounded once, the update relative to p
            close(torch.cat([t.double() for t in got]), torch.cat([w[i] for w in want]), 8 * U[torch.float32] if i or dtype == torch.float32 else U[dtype])


def test_adamw_matches_torch():
    from hive_neuralnet_b200 import train_ops as ops
    torch.manual_seed(0)
    mine = [torch.randn(s, device="cuda") for s in ((7, 5), (300,), (64, 64), (1,))]
    theirs = [p.double().clone().requires_grad_() for p in mine]
    for p in mine:
        p.requires_grad_()
    opt = ops.AdamW(mine, lr=1e-2, betas=(0.8, 0.99), weight_decay=0.1)
    other = torch.optim.AdamW(theirs, lr=1e-2, betas=(0.8, 0.99), weight_decay=0.1)
    for _ in range(20):
        for a, b in zip(mine, theirs):
            b.grad = torch.randn_like(b)
            a.grad = b.grad.float()
        opt.step()
        other.step()
    for a, b in zip(mine, theirs):
        close(a.detach(), b.detach(), 1e-5)  # 20 steps of some ulps


def test_adamw_unaligned_and_strided():
    from hive_neuralnet_b200 import train_ops as ops
    base = torch.randn(2000, device="cuda")
    gbase = torch.randn(2000, device="cuda")
    cut = [base[1:700], base[703:1500]]
    grads = [gbase[2:701], gbase[3:1600:2][:797]]
    whole = [t.clone() for t in cut]
    edge = base.clone()
    m, v = (torch.zeros(ops.state_size(cut), device="cuda") for _ in range(2))
    m2, v2 = m.clone(), v.clone()
    ops.adamw_step(cut, grads, m, v, step=1, **HYPER)
    ops.adamw_step(whole, [g.contiguous().clone() for g in grads], m2, v2, step=1, **HYPER)
    assert torch.equal(m, m2) and torch.equal(v, v2)
    assert all(torch.equal(a, b) for a, b in zip(cut, whole))
    outside = torch.ones(2000, dtype=torch.bool)
    outside[1:700] = outside[703:1500] = False
    assert torch.equal(base.cpu()[outside], edge.cpu()[outside])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [100, 256, 1000, 77_777]])
def test_adamw_8_bits(sizes, dtype):
    """A step from 8-bit states: the parameters as from the values that the codes stand for; the new
    codes are one of the two neighbours of the exact value, and their mean over seeds is that value."""
    from hive_neuralnet_b200 import train_ops as ops
    g = torch.Generator("cuda").manual_seed(9)
    params = [torch.randn(n, generator=g, device="cuda").to(dtype) for n in sizes]
    size = ops.state_size(params)
    codes = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = tuple(torch.zeros(size // 256, device="cuda") for _ in range(2))
    table = [ref.code_values(s).cuda() for s in (False, True)]
    for step in (1, 2, 3):
        grads = [(0.1 * torch.randn(n, generator=g, device="cuda")).to(dtype) for n in sizes]
        m = ops.exp_avg_values(codes[0], scales[0])
        v = ops.exp_avg_sq_values(codes[1], scales[1])
        close(m, table[0][codes[0].long()] * scales[0].double().repeat_interleave(256), 1e-6)
        close(v, (table[1][codes[1].long()] * scales[1].double().repeat_interleave(256)).square(), 1e-6)
        before = [p.clone() for p in params]
        ops.adamw_step(params, grads, *codes, step=step, scales=scales, seed=4, **HYPER)
        ms, vs = [], []
        for p, old, gr, a, b in zip(params, before, grads, parts(m, params), parts(v, params)):
            wp, wm, wv = ref.adamw(old, gr, a, b, step, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
            close(p, wp, 8 * U[torch.float32] if dtype == torch.float32 else U[dtype])
            ms.append(wm)
            vs.append(wv)
        for which, want in ((0, ms), (1, [x.sqrt() for x in vs])):
            for got, w, peak in zip(parts(codes[which], params), want, parts(scales[which].repeat_interleave(256), params)):
                value = table[which][got.long()] * peak.double()
                # a code's spacing: 1/8 (1/16) of its binade, or that of the smallest binade
                gap = torch.maximum(w.abs() * (1 / 8 if which == 0 else 1 / 16), peak.double() * 2.0 ** (-9 if which == 0 else -10))
                assert ((value - w).abs() <= gap * (1 + 1e-5)).all()
                if which:
                    assert (value[w > 0] > 0).all()  # never rounded to none
        for which in (0, 1):  # the gaps between tensors stay empty
            used = torch.zeros(size, dtype=torch.bool, device="cuda")
            for x in parts(used, params):
                x.fill_(True)
            assert not codes[which][~used].any()


def test_adamw_8_bit_rounding_is_unbiased():
    """One value, many positions: the mean of the rounded moments over 2^16 draws is the value, to 5
    standard errors (a code's spacing is at most 1/8 of the value: sd at most 1/16)."""
    from hive_neuralnet_b200 import train_ops as ops
    n = 1 << 16
    p = [torch.zeros(n, device="cuda")]
    g = [torch.full((n,), 0.0137, device="cuda")]
    g[0][::256] = 0.05  # sets the blocks' scale
    codes = [torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = tuple(torch.zeros(n // 256, device="cuda") for _ in range(2))
    ops.adamw_step(p, g, *codes, step=1, scales=scales, seed=1, **HYPER)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[::256] = False
    m = ops.exp_avg_values(codes[0], scales[0])[keep].double()
    r = ops.exp_avg_sq_values(codes[1], scales[1])[keep].double().sqrt()
    tolerance = 5 / 16 / math.sqrt(keep.sum().item())
    assert abs(m.mean().item() / (0.1 * 0.0137) - 1) < tolerance
    assert abs(r.mean().item() / (math.sqrt(0.005) * 0.0137) - 1) < tolerance
    assert len(m.unique()) == 2 and len(r.unique()) == 2
    again = [torch.zeros_like(c) for c in codes]
    ops.adamw_step([torch.zeros(n, device="cuda")], g, *again, step=1, scales=tuple(torch.zeros_like(s) for s in scales), seed=1,
                   **HYPER)
    assert all(torch.equal(a, b) for a, b in zip(again, codes))
    other = [torch.zeros_like(c) for c in codes]
    ops.adamw_step([torch.zeros(n, device="cuda")], g, *other, step=1, scales=tuple(torch.zeros_like(s) for s in scales), seed=2,
                   **HYPER)
    assert not torch.equal(other[0], codes[0])


def test_adamw_8_bit_moments_follow():
    """Constant gradient size for 3000 steps of beta2 = 0.999: the second moment reaches g^2 (nearest
    rounding would stop it after a few steps).  Mean over 4096 values; each is a random walk of codes
    with a spread of about 10 %, so the mean's is 0.2 %, and E[r^2] exceeds E[r]^2 by 1 %: 5 %."""
    from hive_neuralnet_b200 import train_ops as ops
    p = torch.zeros(4096, device="cuda", requires_grad=True)
    opt = ops.AdamW([p], lr=1e-4, state_bits=8, weight_decay=0.0)
    sign = torch.randn(4096, device="cuda").sign()
    for i in range(3000):
        p.grad = 0.01 * sign
        opt.step()
    v = ops.exp_avg_sq_values(opt.exp_avg_sq, opt.scales[1])
    m = ops.exp_avg_values(opt.exp_avg, opt.scales[0])
    assert abs(v.mean().item() / (1e-4 * (1 - 0.999 ** 3000)) - 1) < 0.05
    assert abs((m * sign).mean().item() / 0.01 - 1) < 0.05


def test_adamw_zero_gradients_and_state_dict():
    from hive_neuralnet_b200 import train_ops as ops
    for bits in (8, 32):
        p = torch.randn(1000, device="cuda", requires_grad=True)
        old = p.detach().clone()
        opt = ops.AdamW([p], lr=0.1, weight_decay=0.0, state_bits=bits)
        p.grad = torch.zeros_like(p)
        opt.step()
        assert torch.equal(p.detach(), old)
        p.grad = torch.randn_like(p)
        opt.step()
        twin = old.clone().requires_grad_()
        twin.data.copy_(p.data)
        other = ops.AdamW([twin], lr=0.1, weight_decay=0.0, state_bits=bits)
        other.load_state_dict(opt.state_dict())
        twin.grad = p.grad.clone()
        opt.step()
        other.step()
        assert torch.equal(p.detach(), twin.detach()) and torch.equal(opt.exp_avg, other.exp_avg)
        opt.zero_grad()
        with pytest.raises(ValueError):
            opt.step()


def test_adamw_offsets_past_32_bits():
    from hive_neuralnet_b200 import train_ops as ops
    n = 2 ** 31 + 1000
    p = [torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(300, dtype=torch.bfloat16, device="cuda")]
    g = [torch.full_like(t, 0.01) for t in p]
    size = ops.state_size(p)
    codes = [torch.zeros(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = tuple(torch.zeros(size // 256, device="cuda") for _ in range(2))
    ops.adamw_step(p, g, *codes, step=1, scales=scales, lr=1.0, weight_decay=0.0)
    for t in p:
        assert (t[-200:].float() + 1).abs().max().item() < 0.01 and (t[:200].float() + 1).abs().max().item() < 0.01
    assert codes[0][n - 1] > 0 and codes[0][size - 512] > 0
    assert scales[0][-1] > 0 and scales[0][n // 256] > 0


# ---------------------------------------------------------------------------
# the three together
# ---------------------------------------------------------------------------
def test_hybrid_training_step():
    """hybrid_forward against the module (values and every parameter's gradient), and a run of
    hybrid_train_step that lowers its losses; default and large presets."""
    from oracle import oracle as O

    from hive_neuralnet_b200 import train_ops as ops
    from hive_neuralnet_b200.hybrid import HiveHybridGNN, HybridGNNConfig
    from hive_neuralnet_b200.training import build_hybrid_forward_batch, hybrid_forward, hybrid_train_step
    st = torch.from_numpy(O.oracle().generate_positions(77, 0, 128, 100, 7)).cuda()
    batch = build_hybrid_forward_batch(st, 128)
    rf, sf, atr, na, pb, mf = batch
    for config in (HybridGNNConfig(), HybridGNNConfig.large()):
        torch.manual_seed(0)
        net = HiveHybridGNN(config).cuda()
        for t in net.graph_trunk.layers:
            for e in (t.attn.dq_bias, t.attn.dr_bias, t.attn.dz_bias):
                torch.nn.init.normal_(e.weight, std=0.3)
        wide = type(pb)(pb.token_features[..., :config.node_feat_dim], pb.token_q.long(), pb.token_r.long(),
                        pb.token_z.long(), pb.token_mask.bool(), pb.global_features, pb.num_tokens)
        w = torch.randn(sf.shape[0], device="cuda")
        outs = []
        for forward in (net, lambda *a: hybrid_forward(net, *a)):
            net.zero_grad()
            logits, values = forward(rf, sf, atr, na, wide, mf)
            ((logits * w).mean() + values.square().mean()).backward()
            outs.append((logits.detach(), values.detach(), {k: p.grad.clone() for k, p in net.named_parameters() if p.grad is not None}))
        (l0, v0, g0), (l1, v1, g1) = outs
        close(l1, l0, 1e-4)  # two fp32 paths through four or eight blocks
        close(v1, v0, 1e-4)
        total = torch.cat([g.reshape(-1) for g in g0.values()]).norm().item()
        for name, g in g0.items():
            assert (g1[name] - g).norm().item() <= 1e-3 * g.norm().item() + 1e-5 * total, name
        target = torch.zeros(sf.shape[0], device="cuda")
        target[(na.cumsum(0) - na)[na > 0]] = 1.0
        value = torch.where(torch.arange(128, device="cuda") % 2 == 0, 0.5, -0.5)
        used = [p for k, p in net.named_parameters() if k in g0]
        for bits in (32, 8):
            opt = ops.AdamW(used, lr=2e-3, state_bits=bits)
            losses = [sum(hybrid_train_step(net, opt, batch, target, value)).item() for _ in range(12)]
            assert losses[-1] < losses[0], losses
