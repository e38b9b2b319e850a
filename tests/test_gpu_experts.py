"""
The expert-layer operators on device tensors against plain 64-bit implementations: routing and its plan, ragged products in
every type, 8-bit products, the row quantiser, the weighted sum, and all of them as one layer.

Tolerances are bounds, not observations.  A result of type t carries at most half a step, ``finfo(t).eps / 2`` relative.
Sums in float32 of K products x*w: every addition (a tensor-core instruction adds at least 8 products at once and may
truncate where an addition rounds) loses at most 2^-23 of the running magnitude, which S = sum |x||w| bounds, hence
(K / 8 + 32) 2^-23 S.  A float32 operand split into two TF32 numbers is off by 2^-22, and the product of the two small parts
is dropped: 3 * 2^-22 S more.
"""
import subprocess
import sys

import numpy as np
import pytest

from ios.contrib import ios_runtime as rt

pytestmark = pytest.mark.gpu

torch = pytest.importorskip('torch')

F32, F16, BF16, S8 = torch.float32, torch.float16, torch.bfloat16, torch.int8
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


# ---- routing -----------------------------------------------------------------------------------

def route_reference(logits, k, renormalize):
    """Token by token, in 64 bits."""
    a = logits.double().cpu().numpy()
    tokens, experts = a.shape
    chosen = np.full((tokens, k), -1, dtype=np.int64)
    gates = np.zeros((tokens, k))
    pairs = [[] for _ in range(experts)]
    for t in range(tokens):
        able = [e for e in range(experts) if a[t, e] > -np.inf]
        order = sorted(able, key=lambda e: (-a[t, e], e))
        if not order:
            continue
        top = a[t, order[0]]
        term = {e: 1.0 if a[t, e] == top else np.exp(a[t, e] - top) for e in able}
        total = sum(term[e] for e in (order[:k] if renormalize else able))
        for j, e in enumerate(order[:k]):
            chosen[t, j], gates[t, j] = e, term[e] / total
            pairs[e].append((t, j))
    offsets = np.concatenate([[0], np.cumsum([len(p) for p in pairs])])
    rows, slots = np.full(tokens * k, -1), np.full((tokens, k), -1)
    for at, (t, j) in enumerate(p for of_expert in pairs for p in of_expert):
        rows[at], slots[t, j] = t, at
    return chosen, gates, offsets, rows, slots


def check_route(logits, k, renormalize):
    got = rt.route_experts(logits, k, renormalize)
    chosen, gates, offsets, rows, slots = route_reference(logits, k, renormalize)
    for name, value in (('experts', chosen), ('offsets', offsets), ('rows', rows), ('slots', slots)):
        assert np.array_equal(getattr(got, name).cpu().numpy(), value), name
    # the exponent is off by |l - max| 2^-24, the exponential by 2 steps, a sum of n terms by at most 40 roundings (32 in a
    # lane, 5 across the warp), the quotient by one; the logits below stay within 40 of each other where it matters
    assert np.allclose(got.gates.cpu().numpy(), gates, rtol=90 * U, atol=1e-30)


@pytest.mark.parametrize('tokens,experts,k,dtype', [
    (1, 1, 1, F32), (1, 64, 8, BF16), (3, 5, 5, F16), (9, 33, 2, F32), (128, 40, 8, BF16), (129, 40, 8, F16), (40, 1000, 32, BF16), (255, 16, 4, F16),
    (256, 129, 6, F32), (257, 8, 2, BF16), (1000, 60, 4, F32), (5003, 257, 3, F16), (600, 1024, 32, F32)])
@pytest.mark.parametrize('renormalize', [True, False])
def test_route(tokens, experts, k, dtype, renormalize):
    logits = (2 * torch.randn(tokens, experts, generator=generator(tokens + experts), device='cuda')).to(dtype)
    check_route(logits, k, renormalize)


@pytest.mark.parametrize('tokens', [60, 700])
def test_route_ties_masks_and_odd_values(tokens):
    inf, nan = float('inf'), float('nan')
    logits = torch.randint(-2, 3, (tokens, 24), generator=generator(5), device='cuda').float()    # many equal logits
    logits[1] = -inf                                    # nothing to choose
    logits[2, :] = nan
    logits[3, 3:] = -inf                                # fewer than k
    logits[4] = 0.0
    logits[4, ::2] = -0.0                               # the two zeros tie
    logits[5, 7] = nan
    logits[6] = torch.finfo(F32).min                    # the lowest finite value is a value like any other
    logits[7, 4] = inf
    logits[8, 4:7] = inf
    logits[tokens - 1] = -inf
    for renormalize in (True, False):
        check_route(logits, 4, renormalize)
    check_route(logits[:, :8], 8, True)                 # rows 24 apart, all experts chosen


def test_route_with_nothing_to_route():
    empty = rt.route_experts(torch.empty(0, 8, device='cuda'), 2)
    assert empty.offsets.tolist() == [0] * 9 and empty.rows.numel() == 0 and tuple(empty.slots.shape) == (0, 2)
    masked = rt.route_experts(torch.full((300, 8), -float('inf'), device='cuda'), 2)
    assert masked.offsets.tolist() == [0] * 9
    assert (masked.rows == -1).all() and (masked.slots == -1).all() and (masked.gates == 0).all()


# ---- ragged products ---------------------------------------------------------------------------

def act_reference(v, act):
    return {'identity': lambda t: t, 'relu': lambda t: t.clamp(min=0), 'sigmoid': torch.sigmoid, 'tanh': torch.tanh,
            'silu': lambda t: t * torch.sigmoid(t)}[act](v)


def act_error(v, act):
    """Slope bound times the error of the argument comes on top of this error of the function itself: the fast exponential
    is off by 2 + 1.2 |v| steps of 2^-23, a quotient by 2, tanh by 2; relu and identity are exact."""
    if act in ('identity', 'relu'):
        return torch.zeros_like(v)
    return (6 + 1.2 * v.abs()) * 2.0 ** -23 * act_reference(v, act).abs() + 1e-37


SLOPE = {'identity': 1.0, 'relu': 1.0, 'sigmoid': 0.25, 'tanh': 1.0, 'silu': 1.1}


def grouped_reference(x, weight, bounds, rows=None, bias=None, act='identity', gated=False, row_scale=None,
                      channel_scale=None, out_dtype=None):
    """(value, bound of the error) of every row up to bounds[-1], in 64 bits."""
    total = bounds[-1]
    src = torch.arange(total, device=x.device) if rows is None else rows[:total].long()
    known = (src >= 0) & (src < x.shape[0])
    a = torch.where(known[:, None], x[src.clamp(0, x.shape[0] - 1)].double(), 0.0)
    wide = weight.shape[1]
    v, magnitude = (torch.zeros(total, wide, dtype=torch.float64, device=x.device) for _ in range(2))
    for g in range(weight.shape[0]):
        b, e = bounds[g], bounds[g + 1]
        v[b:e] = a[b:e] @ weight[g].double().t()
        magnitude[b:e] = a[b:e].abs() @ weight[g].double().abs().t()
    group = torch.repeat_interleave(torch.arange(weight.shape[0], device=x.device),
                                    torch.tensor(np.diff(bounds), device=x.device))
    inner = x.shape[1]
    if x.dtype == S8:
        error = U * v.abs()                                # the sum is exact, its conversion rounds
    else:
        error = (inner / 8 + 32) * 2.0 ** -23 * magnitude
        if x.dtype == F32:
            error = error + 3 * 2.0 ** -22 * magnitude
    for scale in (None if row_scale is None else torch.where(known, row_scale[src.clamp(0, x.shape[0] - 1)].double(), 1.0)[:, None],
                  None if channel_scale is None else channel_scale[group].double()):
        if scale is not None:
            v, error = v * scale, error * scale.abs()
            error = error + U * v.abs()
    if bias is not None:
        v = v + bias[group].double()
        error = error + U * v.abs()
    half = wide // 2 if gated else wide
    first, e1 = v[:, :half], error[:, :half]
    value, bound = act_reference(first, act), SLOPE[act] * e1 + act_error(first, act)
    if gated:
        second, e2 = v[:, half:], error[:, half:]
        value, bound = value * second, bound * second.abs() + (value.abs() + bound) * e2 + U * (value * second).abs()
    smallest = torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps
    return value, bound * 1.01 + half_step(out_dtype) * (value.abs() + bound) + smallest


def check_grouped(got, value, bound):
    got = got[:value.shape[0]].double()
    assert torch.isfinite(got).all()
    off = (got - value).abs() - bound
    assert (off <= 0).all(), f'{int((off > 0).sum())} of {off.numel()} beyond the bound, worst by {off.max().item():.3e}'


def make_counts(total, groups, seed, skew=1.0):
    rng = np.random.default_rng(seed)
    shares = rng.permutation((np.arange(groups) + 1.0) ** -skew)
    return np.bincount(rng.choice(groups, size=total, p=shares / shares.sum()), minlength=groups)


def make_operands(gen, shape_x, shape_w, dtype):
    if dtype == S8:
        return (torch.randint(-128, 128, shape_x, generator=gen, device='cuda', dtype=S8),
                torch.randint(-128, 128, shape_w, generator=gen, device='cuda', dtype=S8))
    x = torch.randn(shape_x, generator=gen, device='cuda').to(dtype)
    w = (torch.randn(shape_w, generator=gen, device='cuda') * shape_w[-1] ** -0.5).to(dtype)
    return x, w


def run_grouped(total, groups, inner, channels, dtype, seed=0, gather=False, gated=False, act='identity', bias=False,
                scales=False, out_dtype=None, counts=None, skew=1.0):
    gen = generator(seed + total + inner)
    counts = make_counts(total, groups, seed, skew) if counts is None else np.asarray(counts)
    bounds = np.concatenate([[0], np.cumsum(counts)]).tolist()
    x_rows = max(1, total // 2) if gather else total
    wide = channels * (2 if gated else 1)
    x, w = make_operands(gen, (x_rows, inner), (groups, wide, inner), dtype)
    rows = torch.randint(0, x_rows, (total,), generator=gen, device='cuda', dtype=torch.int32) if gather else None
    args = dict(rows=rows, act=act, gated=gated)
    if bias:
        args['bias'] = torch.randn(groups, wide, generator=gen, device='cuda')
    if scales or dtype == S8:
        size = 1.0 if dtype != S8 else 1.0 / (5000.0 * inner ** 0.5)
        args['row_scale'] = 0.5 + torch.rand(x_rows, generator=gen, device='cuda')
        args['channel_scale'] = size * (0.5 + torch.rand(groups, wide, generator=gen, device='cuda'))
    out_dtype = out_dtype or (BF16 if dtype == S8 else dtype)
    got = rt.grouped_matmul(x, w, torch.tensor(bounds, dtype=torch.int32, device='cuda'), out_dtype=out_dtype, **args)
    assert got.dtype == out_dtype and tuple(got.shape) == (total, channels)
    check_grouped(got, *grouped_reference(x, w, bounds, out_dtype=out_dtype, **args))


ALL_TYPES = pytest.mark.parametrize('dtype', [BF16, F16, F32, S8], ids=['bf16', 'fp16', 'fp32', 'int8'])


@ALL_TYPES
@pytest.mark.parametrize('total,groups,inner,channels', [
    (1, 1, 64, 64), (1, 1, 1, 1), (1, 4, 2048, 512), (8, 64, 512, 320), (33, 3, 96, 130), (100, 7, 17, 33),
    (300, 5, 289, 257), (777, 9, 128, 1000), (1500, 2, 640, 384), (2100, 33, 1024, 192), (64, 2, 4096, 16)])
def test_grouped_product(dtype, total, groups, inner, channels):
    run_grouped(total, groups, inner, channels, dtype)


@ALL_TYPES
@pytest.mark.parametrize('total,groups,inner,channels', [(5, 8, 256, 96), (8, 8, 2048, 512), (30, 3, 1000, 64), (130, 6, 200, 100), (1100, 4, 576, 272), (900, 3, 129, 40)])
def test_grouped_product_gathered_gated(dtype, total, groups, inner, channels):
    run_grouped(total, groups, inner, channels, dtype, gather=True, gated=True, act='silu', bias=True)


@pytest.mark.parametrize('act', ['identity', 'relu', 'sigmoid', 'tanh', 'silu'])
@pytest.mark.parametrize('gated', [False, True])
def test_grouped_product_activations(act, gated):
    run_grouped(150, 4, 192, 72, BF16, act=act, gated=gated, bias=True, scales=True, out_dtype=F32)


@pytest.mark.parametrize('out_dtype', [F32, F16, BF16])
@ALL_TYPES
def test_grouped_product_output_types(dtype, out_dtype):
    run_grouped(90, 4, 128, 136, dtype, bias=True, scales=True, gather=True, out_dtype=out_dtype)


@ALL_TYPES
@pytest.mark.parametrize('counts', [[0, 0, 0, 70], [70, 0, 0, 0], [1, 0, 1, 300], [16, 17, 0, 15], [255, 256, 257, 0], [0, 1, 0, 0]])
def test_grouped_product_uneven_groups(dtype, counts):
    run_grouped(sum(counts), 4, 160, 144, dtype, counts=counts)


# enough rows and channels that two CTAs work on a tile together
@pytest.mark.parametrize('dtype', [BF16, F16, S8], ids=['bf16', 'fp16', 'int8'])
@pytest.mark.parametrize('gather', [False, True])
@pytest.mark.parametrize('counts,inner,channels', [
    ([1700, 0, 3300], 192, 1100), ([256, 4097, 1, 31, 33, 600], 72, 1300), ([5000], 1000, 1030), ([130] * 40, 64, 513)])
def test_grouped_product_in_pairs(dtype, gather, counts, inner, channels):
    run_grouped(sum(counts), len(counts), inner, channels, dtype, counts=counts, gather=gather)
    run_grouped(sum(counts), len(counts), inner, channels, dtype, counts=counts, gather=gather, gated=True, act='silu',
                bias=True, scales=True, out_dtype=F32)


def test_grouped_product_of_many_groups():
    run_grouped(4000, 1024, 64, 48, BF16, skew=0.3)


# few tiles of many columns: the K range split over clusters, few stages
@ALL_TYPES
@pytest.mark.parametrize('gather', [False, True])
@pytest.mark.parametrize('total,groups,inner,channels', [(100, 1, 1024, 64), (128, 1, 2048, 200), (120, 1, 1023, 100), (210, 2, 4000, 130)])
def test_grouped_product_split_over_clusters(dtype, gather, total, groups, inner, channels):
    run_grouped(total, groups, inner, channels, dtype, gather=gather, scales=True, bias=True)
    run_grouped(total, groups, inner, channels, dtype, gather=gather, gated=True, act='silu', out_dtype=F32)


def test_grouped_product_of_many_tiles():
    """More tiles than a CTA finds when it starts: narrow ones, and those of pairs."""
    run_grouped(2000, 1024, 16, 2100, BF16, skew=0.2)
    run_grouped(50000, 2, 8, 5000, BF16, gated=True, skew=0.5)


@ALL_TYPES
def test_grouped_product_strides_and_odd_addresses(dtype):
    """Views into larger buffers: rows apart from one another, first elements at odd addresses, weights of one group shared."""
    gen = generator(3)
    bounds = [0, 40, 40, 131]
    offsets = torch.tensor(bounds, dtype=torch.int32, device='cuda')
    for inner, at, pad in ((128, 0, 16), (128, 1, 7), (70, 2, 10), (63, 1, 0), (130, 0, 1)):
        bx, bw = make_operands(gen, (131, inner + at + pad), (3, 50, inner + at + pad), dtype)
        x, w = bx[:, at:at + inner], bw[:, :, at:at + inner]
        scale = {} if dtype != S8 else {'channel_scale': torch.full((3, 50), 1e-4, device='cuda')}
        whole = torch.full((131, 61), 7.0, dtype=F32, device='cuda')
        out = whole[:, 3:53]
        got = rt.grouped_matmul(x, w, offsets, out=out, **scale)
        assert got.data_ptr() == out.data_ptr()
        check_grouped(got, *grouped_reference(x, w, bounds, out_dtype=F32, **scale))
        assert (whole[:, :3] == 7).all() and (whole[:, 53:] == 7).all()
        shared = w[1:2].expand(3, -1, -1)
        check_grouped(rt.grouped_matmul(x, shared, offsets, out_dtype=F32, **scale),
                      *grouped_reference(x, shared, bounds, out_dtype=F32, **scale))
        same = x[5:6].expand(131, -1)
        check_grouped(rt.grouped_matmul(same, w, offsets, out_dtype=F32, **scale),
                      *grouped_reference(same, w, bounds, out_dtype=F32, **scale))


@ALL_TYPES
@pytest.mark.parametrize('total,stop', [(300, 0), (300, 1), (300, 250), (40, 33)])
def test_rows_behind_the_last_group_are_left(dtype, total, stop):
    gen = generator(total)
    x, w = make_operands(gen, (total, 96), (3, 80, 96), dtype)
    bounds = [0, stop // 3, stop // 2, stop]
    scale = {} if dtype != S8 else {'channel_scale': torch.full((3, 80), 1e-4, device='cuda')}
    if dtype != S8:
        x[stop:] = float('nan')
    out = torch.full((total, 80), 5.0, dtype=BF16, device='cuda')
    rt.grouped_matmul(x, w, torch.tensor(bounds, dtype=torch.int32, device='cuda'), out=out, **scale)
    assert (out[stop:] == 5).all()
    check_grouped(out, *grouped_reference(x[:stop] if stop else x[:0], w, bounds, out_dtype=BF16, **scale)) if stop else None


@ALL_TYPES
def test_rows_that_name_no_row_read_as_zeros(dtype):
    gen = generator(8)
    x, w = make_operands(gen, (20, 64), (2, 40, 64), dtype)
    rows = torch.tensor([3, -1, 19, 20, 0, 2 ** 31 - 1, -2 ** 31, 5, 3], dtype=torch.int32, device='cuda')
    bias = torch.randn(2, 40, generator=gen, device='cuda')
    args = dict(rows=rows, bias=bias, row_scale=torch.rand(20, generator=gen, device='cuda'),
                channel_scale=torch.full((2, 40), 1e-2, device='cuda'))
    got = rt.grouped_matmul(x, w, torch.tensor([0, 4, 9], dtype=torch.int32, device='cuda'), out_dtype=F32, **args)
    check_grouped(got, *grouped_reference(x, w, [0, 4, 9], out_dtype=F32, **args))
    for r in (1, 3):
        assert torch.equal(got[r], bias[0])
    for r in (5, 6):
        assert torch.equal(got[r], bias[1])


@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=['bf16', 'fp16', 'fp32'])
def test_infinities_and_nans_stay_in_their_rows(dtype):
    """Rows of x, also of another group in the same tile, weights of other groups and elements behind a row's end."""
    gen = generator(9)
    bounds = [0, 30, 61, 75]
    offsets = torch.tensor(bounds, dtype=torch.int32, device='cuda')
    buffer, wbuffer = make_operands(gen, (75, 112), (3, 66, 112), dtype)
    buffer[:, 100:] = float('nan')
    wbuffer[:, :, 100:] = float('inf')
    x, w = buffer[:, :100], wbuffer[:, :, :100]
    value, bound = grouped_reference(x, w, bounds, out_dtype=dtype)
    x[31] = float('nan')
    x[60, 3] = float('inf')
    w[2] = float('nan')
    w[1, 5] = float('nan')
    got = rt.grouped_matmul(x, w, offsets)
    keep = torch.ones(75, 66, dtype=torch.bool, device='cuda')
    keep[31], keep[60], keep[61:], keep[30:61, 5] = False, False, False, False
    assert torch.isfinite(got[keep]).all()
    assert ((got.double() - value).abs() <= bound)[keep].all()
    assert torch.isnan(got[31]).all() and torch.isnan(got[61:]).all() and torch.isnan(got[30:61, 5]).all()
    assert not torch.isfinite(got[60]).any()


def test_grouped_product_of_no_rows():
    x = torch.empty(0, 64, dtype=BF16, device='cuda')
    w = torch.randn(3, 8, 64, device='cuda').to(BF16)
    assert tuple(rt.grouped_matmul(x, w, torch.zeros(4, dtype=torch.int32, device='cuda')).shape) == (0, 8)


def test_offsets_that_are_no_plan_stay_inside_the_operands():
    """Decreasing or huge offsets are the caller's mistake: rows get no defined value, but nothing outside is touched."""
    x, w = make_operands(generator(1), (50, 64), (3, 24, 64), BF16)
    whole = torch.full((52, 24), 3.0, dtype=BF16, device='cuda')
    for bad in ([0, 2 ** 31 - 1, 5, 70], [-7, 40, -2 ** 31, 50], [60, 10, 20, 30]):
        rt.grouped_matmul(x, w, torch.tensor(bad, dtype=torch.int32, device='cuda'), out=whole[1:51])
        assert (whole[0] == 3).all() and (whole[51] == 3).all()


# ---- dense 8-bit products and the quantiser -------------------------------------------------------

@pytest.mark.parametrize('rows,inner,channels', [(1, 1, 1), (1, 4096, 1024), (5, 100, 77), (64, 640, 1500), (129, 33, 128),
                                                 (1000, 512, 300), (600, 2049, 520), (257, 1024, 4096)])
@pytest.mark.parametrize('out_dtype', [F32, F16, BF16])
def test_matmul_int8(rows, inner, channels, out_dtype):
    gen = generator(rows + inner)
    a, b = make_operands(gen, (rows, inner), (1, channels, inner), S8)
    args = dict(row_scale=0.5 + torch.rand(rows, generator=gen, device='cuda'),
                channel_scale=(0.5 + torch.rand(channels, generator=gen, device='cuda')) / (5000.0 * inner ** 0.5),
                bias=torch.randn(channels, generator=gen, device='cuda'), act='silu')
    got = rt.matmul_int8(a, b[0], out_dtype=out_dtype, **args)
    reference = dict(args, channel_scale=args['channel_scale'][None], bias=args['bias'][None])
    check_grouped(got, *grouped_reference(a, b, [0, rows], out_dtype=out_dtype, **reference))


def test_matmul_int8_sums_are_exact():
    """Sums past 24 bits whose low bits matter: the largest magnitudes over the longest rows, less one product."""
    for inner in (4096, 131071):
        a = torch.full((3, inner), -128, dtype=S8, device='cuda')
        b = torch.full((40, inner), -128, dtype=S8, device='cuda')
        b[:, -1] = torch.arange(-20, 20, device='cuda').to(S8)
        a[1, -1], a[2, -1] = 1, 0
        expect = (a.double() @ b.double().t())
        base = expect[2, 0].item()
        got = rt.matmul_int8(a, b, bias=torch.full((40,), -base, device='cuda'), out_dtype=F32).double()
        # float32 holds the sum to 2^-24: the difference is right to that
        assert ((got - (expect - base)).abs() <= U * expect.abs()).all()
        small = rt.matmul_int8(a[:, -4:], b[:, -4:], out_dtype=F32).double()
        assert torch.equal(small, a[:, -4:].double() @ b[:, -4:].double().t())


def quantize_reference(x):
    a = x.double()
    finite = torch.isfinite(a)
    largest = torch.where(finite, a.abs(), 0.0).amax(1)
    q = torch.where(finite, torch.round(127.0 * a / torch.where(largest > 0, largest, 1.0)[:, None]), 0.0)
    q = torch.where(torch.isinf(a), 127.0 * torch.sign(a), q)
    return q, largest / 127.0


@pytest.mark.parametrize('dtype', [F32, F16, BF16], ids=['fp32', 'fp16', 'bf16'])
@pytest.mark.parametrize('rows,inner', [(1, 1), (1, 4096), (3, 7), (70, 64), (33, 1000), (9, 12345), (2000, 129), (5, 40000)])
def test_quantize_rows(dtype, rows, inner):
    gen = generator(rows + inner)
    x = torch.randn(rows, inner, generator=gen, device='cuda') * torch.exp(4 * torch.randn(rows, 1, generator=gen, device='cuda'))
    x = x.to(dtype)
    q, scale = rt.quantize_rows(x)
    expect_q, expect_scale = quantize_reference(x)
    assert torch.equal(q.double(), expect_q)
    assert ((scale.double() - expect_scale).abs() <= U * expect_scale + 2.0 ** -150).all()
    at = torch.randint(0, rows, (2 * rows + 1,), generator=gen, device='cuda', dtype=torch.int32)
    q2, scale2 = rt.quantize_rows(x, rows=at)
    assert torch.equal(q2, q[at.long()]) and torch.equal(scale2, scale[at.long()])


@pytest.mark.parametrize('dtype', [F32, F16, BF16], ids=['fp32', 'fp16', 'bf16'])
def test_quantize_rows_ties_and_odd_values(dtype):
    inf, nan, tiny = float('inf'), float('nan'), torch.finfo(dtype).smallest_normal
    x = torch.zeros(12, 40, device='cuda')
    x[0, :20] = torch.arange(20, device='cuda') + 0.5           # halves between whole numbers, with 127 as the largest
    x[0, 30] = 127.0
    x[1, :20] = -(torch.arange(20, device='cuda') + 0.5)
    x[1, 30] = -127.0
    x[2, 0], x[2, 1], x[2, 2] = 3.0, 1.5, -1.5                  # half of the largest: 63.5 rounds to 64
    x[4, 3], x[4, 4], x[4, 5], x[4, 6] = nan, inf, -inf, 2.0
    x[5] = nan
    x[6, 7] = inf
    x[7] = tiny * torch.randn(40, generator=generator(2), device='cuda')
    x[8, 3] = torch.finfo(dtype).max
    x[8, 4] = torch.finfo(dtype).max / 3
    x[9] = -0.0
    x[10] = torch.randn(40, generator=generator(3), device='cuda')
    x[11, 0], x[11, 1] = tiny, 0.5 * tiny
    x = x.to(dtype)
    q, scale = rt.quantize_rows(x)
    expect_q, expect_scale = quantize_reference(x)
    assert torch.equal(q.double(), expect_q)
    assert ((scale.double() - expect_scale).abs() <= U * expect_scale + 2.0 ** -150).all()
    view = torch.cat([x, x], 1)[:, 3:3 + 40]                    # odd addresses, rows apart
    q2, _ = rt.quantize_rows(view)
    assert torch.equal(q2.double(), quantize_reference(view)[0])
    missing, none = rt.quantize_rows(x, rows=torch.tensor([-1, 12, 2], dtype=torch.int32, device='cuda'))
    assert (missing[:2] == 0).all() and (none[:2] == 0).all() and torch.equal(missing[2], q[2])


def test_a_float_between_two_halves_is_not_rounded_twice():
    """float32 values one step off a half: the quotient in float32 would land on it."""
    largest = torch.tensor(1.7, device='cuda')
    steps = torch.arange(0, 127, device='cuda').double() + 0.5
    near = (steps * largest.double() / 127.0).float()
    x = torch.stack([torch.nextafter(near, torch.tensor(0.0, device='cuda')), near, torch.nextafter(near, torch.tensor(9.0, device='cuda'))])
    x = torch.cat([x, largest.expand(3, 1)], 1)
    assert torch.equal(rt.quantize_rows(x)[0].double(), quantize_reference(x)[0])


# ---- weighted sum ---------------------------------------------------------------------------------

@pytest.mark.parametrize('dtype', [F32, F16, BF16], ids=['fp32', 'fp16', 'bf16'])
@pytest.mark.parametrize('tokens,k,channels', [(1, 1, 1), (1, 8, 2048), (7, 3, 77), (300, 2, 1000), (129, 32, 64), (2000, 8, 33)])
def test_combine(dtype, tokens, k, channels):
    gen = generator(tokens + k)
    rows = max(1, tokens * k - 3)
    y = torch.randn(rows, channels, generator=gen, device='cuda').to(dtype)
    gates = torch.randn(tokens, k, generator=gen, device='cuda')
    slots = torch.randint(-1, rows, (tokens, k), generator=gen, device='cuda', dtype=torch.int32)
    slots[0, 0] = rows                                          # beyond the rows: nothing
    if tokens > 1:
        slots[1] = -1
    live = ((slots >= 0) & (slots < rows))[:, :, None]
    parts = torch.where(live, y[slots.clamp(0, rows - 1).long()].double() * gates.double()[:, :, None], 0.0)
    for out_dtype in (dtype, F32):
        got = rt.combine_experts(y, gates, slots, out_dtype=out_dtype).double()
        bound = (k + 1) * U * parts.abs().sum(1)
        bound = 1.01 * bound + half_step(out_dtype) * (parts.sum(1).abs() + bound) + 1e-38 + torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps
        assert ((got - parts.sum(1)).abs() <= bound).all()


def test_combine_views_and_masked_rows():
    gen = generator(4)
    y = torch.randn(50, 90, generator=gen, device='cuda').to(BF16)[:, 5:70]
    y[7] = float('nan')                                          # a row that no slot names
    slots = torch.tensor([[0, 1], [-1, 3], [-1, -1]], dtype=torch.int32, device='cuda')
    gates = torch.tensor([[0.5, 0.25], [float('nan'), 1.0], [float('nan'), 0.0]], device='cuda')
    whole = torch.full((3, 80), 9.0, device='cuda')
    rt.combine_experts(y, gates, slots, out=whole[:, 1:66])
    expect = torch.stack([0.5 * y[0].double() + 0.25 * y[1].double(), y[3].double(), torch.zeros_like(y[0]).double()])
    assert ((whole[:, 1:66].double() - expect).abs() <= 3 * U * (y[0].double().abs() + y[1].double().abs() + y[3].double().abs())).all()
    assert (whole[:, 0] == 9).all() and (whole[:, 66:] == 9).all()
    assert tuple(rt.combine_experts(y, gates[:0], slots[:0]).shape) == (0, 65)
    nothing = rt.combine_experts(y[:0], gates, torch.full_like(slots, -1))
    assert (nothing == 0).all()


# ---- the layer ------------------------------------------------------------------------------------

def layer(x, logits, w_in, w_out, k):
    plan = rt.route_experts(logits, k)
    h = rt.grouped_matmul(x, w_in, plan.offsets, rows=plan.rows, act='silu', gated=True)
    y = rt.grouped_matmul(h, w_out, plan.offsets)
    return rt.combine_experts(y, plan.gates, plan.slots)


def layer_int8(x, logits, w_in, s_in, w_out, s_out, k):
    plan = rt.route_experts(logits, k)
    q, scale = rt.quantize_rows(x)
    h = rt.grouped_matmul(q, w_in, plan.offsets, rows=plan.rows, act='silu', gated=True, row_scale=scale, channel_scale=s_in)
    q, scale = rt.quantize_rows(h)
    y = rt.grouped_matmul(q, w_out, plan.offsets, row_scale=scale, channel_scale=s_out)
    return rt.combine_experts(y, plan.gates, plan.slots, out_dtype=x.dtype)


def layer_reference(x, logits, w_in, w_out, k):
    """Expert by expert over all tokens, in 64 bits, and S = the same with magnitudes."""
    chosen, gates, _, _, _ = route_reference(logits, k, True)
    share = torch.zeros(x.shape[0], w_in.shape[0], dtype=torch.float64)
    for t in range(x.shape[0]):
        for e, g in zip(chosen[t], gates[t]):
            if e >= 0:
                share[t, e] = g
    share = share.cuda()
    out = torch.zeros(x.shape[0], w_out.shape[1], dtype=torch.float64, device='cuda')
    size = torch.zeros_like(out)
    for e in range(w_in.shape[0]):
        gate, up = (x.double() @ w_in[e].double().t()).chunk(2, 1)
        h = gate * torch.sigmoid(gate) * up
        out += share[:, e:e + 1] * (h @ w_out[e].double().t())
        # how far an error of the two products moves h: the gate's slope is at most 1.1
        around = 1.1 * gate.abs() * up.abs() + h.abs()
        size += share[:, e:e + 1] * (around @ w_out[e].double().abs().t())
    return out, size


@pytest.mark.parametrize('tokens,experts,k,inner,outer', [(1, 8, 2, 128, 64), (3, 16, 4, 256, 96), (200, 8, 2, 192, 160), (700, 12, 3, 320, 200)])
@pytest.mark.parametrize('dtype', [BF16, F16, F32], ids=['bf16', 'fp16', 'fp32'])
def test_layer(dtype, tokens, experts, k, inner, outer):
    gen = generator(tokens)
    x = torch.randn(tokens, inner, generator=gen, device='cuda').to(dtype)
    logits = torch.randn(tokens, experts, generator=gen, device='cuda')
    if tokens > 1:
        logits[1] = -float('inf')                               # a padding token
    w_in = (torch.randn(experts, 2 * outer, inner, generator=gen, device='cuda') * inner ** -0.5).to(dtype)
    w_out = (torch.randn(experts, inner, outer, generator=gen, device='cuda') * outer ** -0.5).to(dtype)
    got = layer(x, logits, w_in, w_out, k)
    value, size = layer_reference(x, logits, w_in, w_out, k)
    # three results are rounded to the type (h, y, out), the first product's float32 sums move h by a few steps of 2^-20
    assert ((got.double() - value).abs() <= (3.1 * half_step(dtype) + 2.0 ** -16) * size + 1e-6).all()
    if tokens > 1:
        assert (got[1] == 0).all()
    again = layer(x, logits, w_in, w_out, k)
    assert torch.equal(got, again)                              # the same bits every time


def test_layer_in_8_bits():
    gen = generator(77)
    tokens, experts, k, inner, outer = 150, 8, 2, 256, 192
    x = torch.randn(tokens, inner, generator=gen, device='cuda').to(BF16)
    logits = torch.randn(tokens, experts, generator=gen, device='cuda')
    w_in = torch.randn(experts, 2 * outer, inner, generator=gen, device='cuda') * inner ** -0.5
    w_out = torch.randn(experts, inner, outer, generator=gen, device='cuda') * outer ** -0.5
    (q_in, s_in), (q_out, s_out) = (rt.quantize_rows(w.flatten(0, 1)) for w in (w_in, w_out))
    q_in, s_in = q_in.view_as(w_in), s_in.view(w_in.shape[:2])
    q_out, s_out = q_out.view_as(w_out), s_out.view(w_out.shape[:2])
    got = layer_int8(x, logits, q_in, s_in, q_out, s_out, k)
    # against the same layer with the weights that the integers stand for and the tokens rounded to 8 bits
    q, scale = rt.quantize_rows(x)
    value, _ = layer_reference(q.double() * scale.double()[:, None], logits, q_in.double() * s_in.double()[:, :, None],
                               q_out.double() * s_out.double()[:, :, None], k)
    # h is rounded to 8 bits: at most half a step of its row's largest / 127, in the root mean square over a row of normal
    # products far below 1 / 50 of the result's size
    assert (got.double() - value).norm() <= 0.02 * value.norm()


def test_elements_past_32_bits():
    """Matrices of more than 2^31 elements: the product's result, the quantiser's and the weighted sum's input."""
    gen = generator(12)
    rows, channels, inner = 540000, 4096, 16
    x, w = make_operands(gen, (rows, inner), (2, channels, inner), BF16)
    bounds = [0, 1000, rows]
    y = rt.grouped_matmul(x, w, torch.tensor(bounds, dtype=torch.int32, device='cuda'))
    assert y.numel() > 2 ** 31
    tail = slice(rows - 300, rows)
    check_grouped(y[tail], *grouped_reference(x[tail], w[1:], [0, 300], out_dtype=BF16))
    check_grouped(y[:300], *grouped_reference(x[:300], w[:1], [0, 300], out_dtype=BF16))
    q, scale = rt.quantize_rows(y)
    expect, expect_scale = quantize_reference(y[tail])
    assert torch.equal(q[tail].double(), expect)
    assert ((scale[tail].double() - expect_scale).abs() <= U * expect_scale).all()
    slots = torch.tensor([[rows - 1, rows - 2], [0, rows - 300]], dtype=torch.int32, device='cuda')
    gates = torch.tensor([[0.5, 0.25], [2.0, 1.0]], device='cuda')
    got = rt.combine_experts(y, gates, slots, out_dtype=F32).double()
    parts = y[slots.long()].double() * gates.double()[:, :, None]
    assert ((got - parts.sum(1)).abs() <= 3 * U * parts.abs().sum(1)).all()
    again = rt.grouped_matmul(q, torch.ones(1, 8, channels, dtype=S8, device='cuda'), torch.tensor([0, rows], dtype=torch.int32, device='cuda'),
                              row_scale=scale, out_dtype=F32)
    assert torch.allclose(again[tail, 0].double(), q[tail].double().sum(1) * scale[tail].double(), rtol=4 * U)


def test_captured_layer_on_a_side_stream_with_new_inputs():
    """A layer captured into a graph follows its inputs; two graphs and an eager call run at once."""
    gen = generator(6)
    tokens, experts, k, inner, outer = 300, 8, 2, 128, 96
    w_in = (torch.randn(experts, 2 * outer, inner, generator=gen, device='cuda') * inner ** -0.5).to(BF16)
    w_out = (torch.randn(experts, inner, outer, generator=gen, device='cuda') * outer ** -0.5).to(BF16)
    sets = [(torch.randn(tokens, inner, generator=gen, device='cuda').to(BF16), torch.randn(tokens, experts, generator=gen, device='cuda'))
            for _ in range(5)]
    expect = [layer(x, l, w_in, w_out, k) for x, l in sets]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        x, l = (t.clone() for t in sets[i])
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            layer(x, l, w_in, w_out, k)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = layer(x, l, w_in, w_out, k)
        graphs.append((graph, x, l, out, stream))
    for j in (2, 3, 4):
        for graph, x, l, out, stream in graphs:
            with torch.cuda.stream(stream):
                x.copy_(sets[j][0])
                l.copy_(sets[j][1])
                graph.replay()
        eager = layer(*sets[j], w_in, w_out, k)
        torch.cuda.synchronize()
        assert torch.equal(eager, expect[j])
        for _, _, _, out, _ in graphs:
            assert torch.equal(out, expect[j])


def test_the_first_call_of_a_process_may_be_a_captured_one():
    code = '''
import sys
sys.path[:0] = %r
import torch
from test_gpu_experts import layer
from ios.contrib import ios_runtime as rt
x, logits = torch.randn(20, 64, device="cuda").bfloat16(), torch.randn(20, 4, device="cuda")
w_in, w_out = torch.randn(4, 96, 64, device="cuda").bfloat16(), torch.randn(4, 64, 48, device="cuda").bfloat16()
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    out = layer(x, logits, w_in, w_out, 2)
graph.replay()
assert torch.equal(out, layer(x, logits, w_in, w_out, 2))
rt.device_ops_status()
''' % [path for path in sys.path if path]
    done = subprocess.run([sys.executable, '-c', code], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


def test_no_wait_ran_out():
    rt.device_ops_status()


def test_the_current_device_is_left_alone_and_host_memory_refused():
    before = torch.cuda.current_device()
    x = torch.randn(4, 8, device='cuda')
    rt.quantize_rows(x)
    assert torch.cuda.current_device() == before
    host = torch.zeros(4, 8)
    q, s = torch.empty(4, 8, dtype=S8, device='cuda'), torch.empty(4, device='cuda')
    lib = rt._library()
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.ios_quantize_rows(host.data_ptr(), 0, 4, 8, 8, None, 4, q.data_ptr(), 8, s.data_ptr(), stream) == 3
    assert b'device memory' in lib.ios_last_error()
    assert lib.ios_quantize_rows(x.data_ptr(), 0, 4, 8, 8, None, 4, host.data_ptr(), 8, s.data_ptr(), stream) == 3
    with pytest.raises(ValueError, match='gradient'):
        rt.quantize_rows(x.clone().requires_grad_())
    with torch.no_grad():
        rt.quantize_rows(x.clone().requires_grad_())
    with pytest.raises(ValueError, match='dense'):
        rt.quantize_rows(torch.randn(8, 4, device='cuda').t())
    with pytest.raises(ValueError, match='one type'):
        rt.grouped_matmul(x, torch.zeros(1, 4, 8, dtype=BF16, device='cuda'), torch.zeros(2, dtype=torch.int32, device='cuda'))
