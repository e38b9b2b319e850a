"""
Calls of the expert-layer operators at the edges of what they take: huge magnitudes, sizes next to a launch limit, several
host threads, row counts past a limit, waits that run out.  References and tolerances as in test_gpu_experts.py.
"""
import subprocess
import sys
import threading

import pytest

from ios.contrib import ios_runtime as rt

pytestmark = pytest.mark.gpu

torch = pytest.importorskip('torch')

from test_gpu_experts import BF16, F16, F32, S8, U, check_route, generator, half_step, layer, make_operands, quantize_reference  # noqa: E402


# ---- quantiser: magnitudes whose products with 254 pass float32 ------------------------------------

def rows_of_halves(power, width, dtype):
    """All halves n + 1/2 below 127 of a row whose largest is 127, both signs, times a power of two: exact in every type."""
    halves = torch.arange(127, device='cuda').double() + 0.5
    row = torch.cat([halves, torch.tensor([127.0], dtype=torch.float64, device='cuda')]) * 2.0 ** power
    return torch.stack([row, -row]).repeat(1, width // 128).to(dtype)


@pytest.mark.parametrize('dtype', [BF16, F32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('power', [121, 120, 118, 93, 92, 0, -107, -108, -126])
@pytest.mark.parametrize('width', [128, 2048, 4096, 8192])
def test_quantized_halves_at_any_magnitude(dtype, power, width):
    x = rows_of_halves(power, width, dtype)
    q, scale = rt.quantize_rows(x)
    expect, expect_scale = quantize_reference(x)
    assert torch.equal(q.double(), expect)
    assert ((scale.double() - expect_scale).abs() <= U * expect_scale + 2.0 ** -150).all()
    odd = torch.cat([x, x], 1)[:, 1:width + 1]                  # element by element
    assert torch.equal(rt.quantize_rows(odd)[0].double(), quantize_reference(odd)[0])


@pytest.mark.parametrize('dtype', [F16, BF16, F32], ids=['fp16', 'bf16', 'fp32'])
def test_quantized_rows_of_huge_values(dtype):
    top = torch.finfo(dtype).max
    x = (torch.randn(200, 1000, generator=generator(21), device='cuda') * (top / 6)).clamp(-top, top).to(dtype)
    x[0, :3] = torch.tensor([top, top / 2, -top], device='cuda').to(dtype)
    x[1, 5], x[2, 6] = float('inf'), float('nan')
    for view in (x, x[:, 1:]):
        assert torch.equal(rt.quantize_rows(view)[0].double(), quantize_reference(view)[0])


# ---- router: shared memory next to the default limit, several host threads -----------------------------

@pytest.mark.parametrize('tokens,experts,k', [(108, 320, 8), (42, 352, 8), (120, 256, 16), (128, 1024, 32), (129, 1024, 32)])
def test_first_route_of_a_process_at_any_size(tokens, experts, k):
    """The first three need 48 KiB of shared memory with the kernel's own arrays, and less without; each is the first call."""
    code = '''
import sys
sys.path[:0] = %r
import torch
from test_gpu_experts import check_route
check_route(torch.randn(%d, %d, device="cuda"), %d, True)
''' % ([path for path in sys.path if path], tokens, experts, k)
    done = subprocess.run([sys.executable, '-c', code], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr[-2000:]


def test_route_from_several_host_threads():
    """Calls of one kernel with different shared-memory sizes, from threads that do not wait for one another."""
    shapes = [(600, 1024, 8), (4000, 520, 8), (600, 520, 2), (300, 1000, 32)]
    inputs = [torch.randn(t, e, generator=generator(t + e), device='cuda') for t, e, _ in shapes]
    expect = [rt.route_experts(l, k) for l, (_, _, k) in zip(inputs, shapes)]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(1500):
                    got = rt.route_experts(inputs[i], shapes[i][2])
                torch.cuda.current_stream().synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, expect[i]))
        except Exception as error:
            failed.append((shapes[i], error))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(shapes))]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failed, failed


# ---- products whose waits run out -------------------------------------------------------------------

@pytest.fixture
def short_waits():
    """Sets what a wait inside a product may take, in microseconds; the default comes back, and the record is read, at the end."""
    yield lambda us: rt.set_option('product_wait_us', us)
    rt.set_option('product_wait_us', 0)
    try:
        rt.device_ops_status()
    except RuntimeError:
        pass


def ran_out():
    try:
        rt.device_ops_status()
    except RuntimeError as error:
        assert 'ran out' in str(error)
        return True
    return False


def test_a_wait_that_runs_out_is_reported_and_ends(short_waits):
    """One tile whose sums take far longer than its epilogue may wait: the rest of the product ends by itself."""
    inner = 1 << 23
    x = torch.ones(1, inner, dtype=BF16, device='cuda').expand(64, -1)
    w = torch.ones(1, 1, inner, dtype=BF16, device='cuda').expand(1, 128, -1)
    offsets = torch.tensor([0, 64], dtype=torch.int32, device='cuda')
    scale = torch.ones(64, device='cuda')
    short_waits(100)
    rt.grouped_matmul(x, w, offsets, row_scale=scale)
    assert ran_out()
    short_waits(0)
    small = rt.grouped_matmul(x[:, :4096], w[:, :, :4096], offsets, row_scale=scale)
    assert (small == 4096).all()
    assert not ran_out()


@pytest.mark.parametrize('us', [100, 1500, 6000])
@pytest.mark.parametrize('dtype,x_rows,total,inner,channels,gather', [
    (BF16, 1, 6000, 1 << 20, 1500, False), (BF16, 256, 12000, 1 << 20, 1024, True), (BF16, 100, 100, 1 << 22, 128, False),
    (F32, 2000, 2000, 1 << 18, 1500, False)], ids=['loaders', 'gathered-pairs', 'cluster', 'float'])
def test_products_end_whichever_wait_runs_out(short_waits, us, dtype, x_rows, total, inner, channels, gather):
    """Tiles of a millisecond or more, several per CTA, and scales that the epilogue warps share: some waits run out and some do
    not, every kernel returns, and the next one is whole."""
    gen = generator(total)
    x = torch.empty(x_rows, inner, dtype=dtype, device='cuda').uniform_(-1, 1, generator=gen)
    w = torch.empty(1, 1 if x_rows == 1 else channels, inner, dtype=dtype, device='cuda').uniform_(-1, 1, generator=gen)
    if x_rows == 1:
        x, w = x.expand(total, -1), w.expand(1, channels, -1)
    args = dict(row_scale=torch.rand(x.shape[0], generator=gen, device='cuda'), out_dtype=F32)
    if gather:
        args['rows'] = torch.randint(0, x_rows, (total,), generator=gen, device='cuda', dtype=torch.int32)
    offsets = torch.tensor([0, total], dtype=torch.int32, device='cuda')
    expect = rt.grouped_matmul(x, w, offsets, **args)
    assert not ran_out()
    short_waits(us)
    for _ in range(2):
        got = rt.grouped_matmul(x, w, offsets, **args)
        if not ran_out():
            assert torch.equal(got, expect)
    short_waits(0)
    assert torch.equal(rt.grouped_matmul(x, w, offsets, **args), expect)
    assert not ran_out()


def test_every_thread_is_told_of_a_wait_that_ran_out(short_waits):
    """One thread's question does not answer another's; nobody is told twice."""
    inner = 1 << 23
    x = torch.ones(1, inner, dtype=BF16, device='cuda').expand(64, -1)
    w = torch.ones(1, 1, inner, dtype=BF16, device='cuda').expand(1, 128, -1)
    told, asked = {}, [threading.Barrier(3) for _ in range(3)]

    def ask(name):
        ran_out()                                               # what lies before this test
        asked[0].wait(60)
        asked[1].wait(60)                                       # the product has run out of time meanwhile
        told[name] = (ran_out(), ran_out())
        asked[2].wait(60)

    threads = [threading.Thread(target=ask, args=(name,)) for name in ('first', 'second')]
    for thread in threads:
        thread.start()
    ran_out()
    asked[0].wait(60)
    short_waits(100)
    rt.grouped_matmul(x, w, torch.tensor([0, 64], dtype=torch.int32, device='cuda'))
    assert ran_out() and not ran_out()
    asked[1].wait(60)
    asked[2].wait(60)
    for thread in threads:
        thread.join()
    assert told == {'first': (True, False), 'second': (True, False)}


# ---- router: calls of more blocks than read one another's counts -----------------------------------------

@pytest.mark.parametrize('tokens,experts,k,dtype', [
    (131072, 64, 8, BF16), (131073, 64, 8, BF16), (300000, 100, 32, F32), (1100003, 4, 1, F16), (270000, 1024, 4, F32), (33000, 33, 32, BF16)])
def test_route_of_many_tokens(tokens, experts, k, dtype):
    logits = torch.randn(tokens, experts, generator=generator(tokens), device='cuda').to(dtype)
    logits[::17] = -float('inf')
    got = rt.route_experts(logits, k)
    best, index = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    chosen = torch.where(best[:, :k] > -float('inf'), index[:, :k], -1)
    assert torch.equal(got.experts.long(), chosen)
    flat = torch.where(chosen < 0, experts, chosen).flatten()
    order = torch.sort(flat, stable=True).indices
    counts = torch.bincount(flat, minlength=experts + 1)[:experts]
    used = int(counts.sum())
    assert torch.equal(got.offsets.long(), torch.cat([counts.new_zeros(1), counts.cumsum(0)]))
    assert torch.equal(got.rows[:used].long(), order[:used] // k) and (got.rows[used:] == -1).all()
    slots = torch.full_like(flat, -1)
    slots[order[:used]] = torch.arange(used, device='cuda')
    assert torch.equal(got.slots.flatten().long(), slots)
    gates = torch.softmax(best[:, :k].double(), 1).nan_to_num(0.0)
    assert ((got.gates.double() - gates).abs() <= 90 * U * gates + 1e-30).all()


# ---- activations far from zero ---------------------------------------------------------------------------

@pytest.mark.parametrize('out_dtype', [BF16, F16, F32], ids=['bf16', 'fp16', 'fp32'])
@pytest.mark.parametrize('act', ['silu', 'sigmoid'])
def test_activations_far_from_zero(act, out_dtype):
    """exp(-v) passes float32 below v = -88, the result does not.  The exponential is off by 2 + 1.2 |v| steps of 2^-23, the quotient and
    the product by 3 more; below 2^-126 steps have one size, 2^-149, which |v| <= 104 multiplies."""
    v = torch.cat([torch.arange(-104.0, 20.0, 0.25, device='cuda'), torch.tensor([-1e30, -200.0, 200.0, 1e30, 0.0, -0.0], device='cuda')]).to(BF16)
    got = rt.grouped_matmul(torch.ones(1, 1, dtype=BF16, device='cuda'), v[None, :, None].contiguous(),
                            torch.tensor([0, 1], dtype=torch.int32, device='cuda'), act=act, out_dtype=out_dtype)[0].double()
    a = v.double()
    expect = a * torch.sigmoid(a) if act == 'silu' else torch.sigmoid(a)
    bound = (6 + 1.2 * a.abs().clamp(max=104)) * 2.0 ** -23 * expect.abs() + 2.0 ** -140
    bound = bound + half_step(out_dtype) * (expect.abs() + bound) + torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps
    inside = expect.abs() <= torch.finfo(out_dtype).max
    assert ((got - expect).abs() <= bound)[inside].all()
    special = torch.tensor([float('inf'), float('nan')], device='cuda').to(BF16)
    got = rt.grouped_matmul(torch.ones(1, 1, dtype=BF16, device='cuda'), special[None, :, None].contiguous(),
                            torch.tensor([0, 1], dtype=torch.int32, device='cuda'), act=act, out_dtype=out_dtype)[0]
    assert got[0] == (float('inf') if act == 'silu' else 1.0) and torch.isnan(got[1])


@pytest.mark.parametrize('out_dtype', [BF16, F32], ids=['bf16', 'fp32'])
def test_relu_of_nan_is_zero(out_dtype):
    w = torch.tensor([float('nan'), -1.0, 2.0, float('inf')], device='cuda').to(BF16)[None, :, None]
    got = rt.grouped_matmul(torch.ones(1, 1, dtype=BF16, device='cuda'), w, torch.tensor([0, 1], dtype=torch.int32, device='cuda'), act='relu',
                            out_dtype=out_dtype)
    assert got.tolist() == [[0.0, 0.0, 2.0, float('inf')]]


# ---- sizes past 32 bits ------------------------------------------------------------------------------------

def test_sizes_past_32_bits_are_refused():
    """(A row count of 2^32 + 4 is 4 in 32 bits: the rest of the result would be left unwritten.)"""
    many, offsets = 2 ** 32 + 4, torch.zeros(2, dtype=torch.int32, device='cuda')
    row, row8 = torch.zeros(1, 16, dtype=BF16, device='cuda'), torch.zeros(1, 16, dtype=S8, device='cuda')
    for call in (lambda: rt.route_experts(row.expand(many, -1), 1), lambda: rt.matmul_int8(row8.expand(many, -1), row8),
                 lambda: rt.matmul_int8(row8, row8.expand(many, -1)), lambda: rt.quantize_rows(row.expand(many, -1)),
                 lambda: rt.grouped_matmul(row.expand(many, -1), row[None], offsets),
                 lambda: rt.grouped_matmul(row, row[None].expand(1, many, -1), offsets),
                 lambda: rt.grouped_matmul(row, row[None].expand(many, -1, -1), offsets),
                 lambda: rt.route_experts(row.expand(2 ** 30, -1), 2)):
        with pytest.raises(ValueError, match='more than'):
            call()
    wide = torch.zeros(1, 2 ** 31 + 8, dtype=S8, device='cuda')
    with pytest.raises(ValueError, match='more than'):
        rt.matmul_int8(wide, wide)
    with pytest.raises(ValueError, match='more than'):
        rt.quantize_rows(torch.zeros(1, 2 ** 31, dtype=F16, device='cuda'))


# ---- rows that name none of no rows --------------------------------------------------------------------------

@pytest.mark.parametrize('dtype', [BF16, F16, F32, S8], ids=['bf16', 'fp16', 'fp32', 'int8'])
@pytest.mark.parametrize('gated', [False, True])
def test_product_of_rows_that_are_not_there(dtype, gated):
    """x without rows: every entry of `rows` reads as zeros, whatever the weights hold."""
    gen = generator(5)
    _, w = make_operands(gen, (1, 64), (2, 48, 64), dtype)
    if dtype != S8:
        w[0, 0] = float('nan')
    x, bias = w.new_empty(0, 64), torch.randn(2, 48, generator=gen, device='cuda')
    offsets, rows = (torch.tensor(v, dtype=torch.int32, device='cuda') for v in ([0, 3, 40], [-1, 0, 2 ** 31 - 1] + [-1] * 37))
    got = rt.grouped_matmul(x, w, offsets, rows=rows, bias=bias, act='relu', gated=gated, out_dtype=F32, row_scale=x.new_empty(0, dtype=F32),
                            channel_scale=torch.ones(2, 48, device='cuda'))
    v = torch.repeat_interleave(bias, torch.tensor([3, 37], device='cuda'), 0)
    assert torch.equal(got, v[:, :24].clamp(min=0) * v[:, 24:] if gated else v.clamp(min=0))


@pytest.mark.parametrize('inner', [64, 63])
def test_quantized_rows_that_are_not_there(inner):
    q, scale = rt.quantize_rows(torch.empty(0, inner, device='cuda'), rows=torch.tensor([-1, 0, 5], dtype=torch.int32, device='cuda'))
    assert tuple(q.shape) == (3, inner) and (q == 0).all() and (scale == 0).all()


# ---- derivatives, versions ---------------------------------------------------------------------------------------

def test_tangents_are_refused():
    """Forward-mode derivatives of any argument, also under torch.no_grad(), which does not switch them off."""
    from torch.autograd import forward_ad
    x, w, logits = torch.randn(4, 8, device='cuda'), torch.randn(1, 6, 8, device='cuda'), torch.randn(4, 3, device='cuda')
    offsets, bias = torch.tensor([0, 4], dtype=torch.int32, device='cuda'), torch.randn(1, 6, device='cuda')
    plan = rt.route_experts(logits, 2)
    y = torch.randn(8, 8, device='cuda')
    expect = rt.grouped_matmul(x, w, offsets, bias=bias)
    with forward_ad.dual_level(), torch.no_grad():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: rt.route_experts(dual(logits), 2), lambda: rt.grouped_matmul(dual(x), w, offsets),
                     lambda: rt.grouped_matmul(x, dual(w), offsets), lambda: rt.grouped_matmul(x, w, offsets, bias=dual(bias)),
                     lambda: rt.quantize_rows(dual(x)), lambda: rt.combine_experts(dual(y), plan.gates, plan.slots),
                     lambda: rt.combine_experts(y, dual(plan.gates), plan.slots)):
            with pytest.raises(ValueError, match='tangent'):
                call()
        assert torch.equal(rt.grouped_matmul(forward_ad.unpack_dual(dual(x)).primal, w, offsets, bias=bias), expect)


def test_a_result_written_into_a_saved_tensor_is_noticed():
    """torch refuses a backward pass through a tensor that an `out` has overwritten since."""
    x, w = torch.randn(4, 8, device='cuda'), torch.randn(1, 6, 8, device='cuda')
    offsets = torch.tensor([0, 4], dtype=torch.int32, device='cuda')
    plan = rt.route_experts(torch.randn(4, 3, device='cuda'), 2)
    q = torch.ones(4, 16, dtype=S8, device='cuda')
    for write, shape in ((lambda out: rt.grouped_matmul(x, w, offsets, out=out), (4, 6)), (lambda out: rt.matmul_int8(q, q, out=out), (4, 4)),
                         (lambda out: rt.combine_experts(torch.randn(8, 8, device='cuda'), plan.gates, plan.slots, out=out), (4, 8))):
        leaf, out = torch.ones(shape, device='cuda', requires_grad=True), torch.ones(shape, device='cuda')
        product = (leaf * out).sum()
        write(out)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            product.backward()
    with torch.inference_mode():
        out = torch.empty(4, 6, device='cuda')
        assert torch.equal(rt.grouped_matmul(x, w, offsets, out=out), rt.grouped_matmul(x, w, offsets))


# ---- 8-bit products: sums of 32 bits ------------------------------------------------------------------------------

# few rows (K split over a cluster), tiles of one CTA, pairs of CTAs, rows at odd addresses, the longest rows
@pytest.mark.parametrize('rows,inner,channels', [(3, 4096, 300), (20, 4095, 300), (300, 4096, 1100), (1500, 4096, 2100), (3, 131070, 40), (400, 131071, 40)])
def test_matmul_int8_sums_pass_24_bits(rows, inner, channels):
    """
    Odd products that pass 2^24 and cancel: the result is below 2^24, so float32 holds it exactly, but a float32 sum on the
    way, where only even numbers are left, does not reach it.
    """
    gen, half = generator(inner + rows), inner // 2
    a, b = (torch.randint(50, 64, (n, half), generator=gen, device='cuda', dtype=S8) * 2 + 1 for n in (rows, channels))
    rest = inner - 2 * half
    a = torch.cat([a, -a, torch.ones(rows, rest, dtype=S8, device='cuda')], 1)
    b = torch.cat([b, b, torch.ones(channels, rest, dtype=S8, device='cuda')], 1)
    b[:, inner - 3] -= 3
    expect = a.double() @ b.double().t()
    assert expect.abs().max() < 2 ** 24 and half * 101 ** 2 > 2 ** 24
    in_float32 = (a[0].cpu().float() * b[0].cpu().float()).numpy().cumsum(dtype='float32')[-1]
    assert in_float32 != expect[0, 0].item()
    assert torch.equal(rt.matmul_int8(a, b, out_dtype=F32).double(), expect)


# ---- the longest rows -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize('odd', [0, 1])
def test_the_longest_16_bit_rows_are_summed_in_time(odd):
    """2^25 elements in one CTA each, through the slowest loads: the epilogue waits for all of them at once."""
    inner, channels = (1 << 25) - odd, 128 * 100
    row = torch.ones(1, inner + odd, dtype=BF16, device='cuda')[:, odd:]
    x = torch.ones(1, inner, dtype=BF16, device='cuda').expand(128, -1)
    row[0, 1::2] = -1
    row[0, 7:1001:2] = 1                                        # 497 of them: 994 more, and an odd row has one 1 more than -1
    assert not ran_out()
    got = rt.grouped_matmul(x, row[None].expand(1, channels, -1), torch.tensor([0, 128], dtype=torch.int32, device='cuda'), out_dtype=F32)
    assert not ran_out()
    assert (got == 994 + odd).all()


# ---- float32 elements whose smaller half is subnormal ---------------------------------------------------------------------

@pytest.mark.parametrize('power', [100, 114, 118, 122, 126, 135])
@pytest.mark.parametrize('pad', [0, 1])
def test_float32_products_of_tiny_elements(power, pad):
    """An element split in two loses at most 2^-22 of itself, or 2^-137, half of the last step that its smaller half has."""
    gen = generator(power)
    inner = 200
    x = (torch.randn(70, inner + pad, generator=gen, device='cuda').double() * 2.0 ** -power).float()[:, pad:]
    w = (torch.randn(1, 90, inner + pad, generator=gen, device='cuda').double() * 2.0 ** min(power, 120)).float()[:, :, pad:]
    offsets = torch.tensor([0, 70], dtype=torch.int32, device='cuda')
    got = rt.grouped_matmul(x, w, offsets).double()
    a, b = x.double(), w[0].double()
    size = a.abs() @ b.abs().t()
    bound = (inner / 8 + 32) * 2.0 ** -23 * size + 3 * 2.0 ** -22 * size + 2.0 ** -137 * b.abs().sum(1)[None]
    assert ((got - a @ b.t()).abs() <= 1.01 * bound + 2.0 ** -149).all()


# ---- router: values of 16 bits that are no ordinary numbers ----------------------------------------------------------------

@pytest.mark.parametrize('dtype', [BF16, F16], ids=['bf16', 'fp16'])
@pytest.mark.parametrize('tokens', [60, 700])
def test_route_of_odd_16_bit_values(dtype, tokens):
    inf, nan, info = float('inf'), float('nan'), torch.finfo(dtype)
    logits = torch.randint(-2, 3, (tokens, 40), generator=generator(6), device='cuda').to(dtype)      # many equal logits
    logits[1] = -inf
    logits[2] = nan
    logits[3] = -nan
    logits[4, 2:] = -inf
    logits[5] = 0.0
    logits[5, ::2] = -0.0                               # the two zeros tie
    logits[6] = info.min
    logits[7, 39], logits[7, 5] = inf, info.max
    logits[8, 4:9] = inf
    logits[9, ::3], logits[9, 1::3] = nan, -nan
    logits[10] = torch.arange(40, device='cuda').to(dtype) * info.smallest_normal * info.eps           # subnormal ones have an order, too
    for renormalize in (True, False):
        check_route(logits, 8, renormalize)


# ---- beside the graph path ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('precision', ['tf32x3', 'bf16'])
def test_layers_and_an_engine_at_once(precision):
    """Both use tensor memory and clusters: an engine in one thread, layers on a stream in another, neither changes a bit."""
    import numpy as np
    import ios
    import ios_oracle as oracle
    from helpers import seeded
    rt.set_option('precision', precision)
    try:
        graph = ios.models.inception_v3()
        graph.greedy_schedule()
        config, _ = seeded(graph, 0)
        engine = rt.Engine(graph, 1)
    finally:
        rt.set_option('precision', 'tf32x3')
    image = oracle.normal_input(config, 1, 0)
    expect = engine.run(image)
    gen = generator(31)
    inputs = []
    for tokens, experts, k, inner, outer, dtype in ((4, 16, 4, 1024, 512, BF16), (700, 8, 2, 512, 768, F16), (33, 8, 2, 256, 192, F32)):
        x = torch.randn(tokens, inner, generator=gen, device='cuda').to(dtype)
        w_in = (torch.randn(experts, 2 * outer, inner, generator=gen, device='cuda') * inner ** -0.5).to(dtype)
        w_out = (torch.randn(experts, inner, outer, generator=gen, device='cuda') * outer ** -0.5).to(dtype)
        inputs.append((x, torch.randn(tokens, experts, generator=gen, device='cuda'), w_in, w_out, k))
    alone = [layer(*args) for args in inputs]
    torch.cuda.synchronize()
    failed, done = [], threading.Event()

    def images():
        try:
            for _ in range(150):
                assert np.array_equal(engine.run(image), expect)
        except Exception as error:
            failed.append(error)
        done.set()

    thread = threading.Thread(target=images)
    thread.start()
    with torch.cuda.stream(torch.cuda.Stream()):
        while not done.is_set():
            for args, value in zip(inputs, alone):
                assert torch.equal(layer(*args), value)
    thread.join()
    engine.close()
    assert not failed, failed
    assert not ran_out()
