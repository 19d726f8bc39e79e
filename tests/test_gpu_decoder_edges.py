"""GPU tests of what layer_norm, linear_act_int8 and sample_labels do at their edges: what a kernel keeps between its
passes, settings at the ends of their ranges, logits far from zero, waits that run out in a part of a warp."""
import ctypes

import pytest
import torch

import decoder_lib as dl
import heads_abi as ha
import heads_lib as hl
from test_decoder_cpu import Sampling

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = dict(argvalues=[F32, F16, BF16], ids=["f32", "f16", "bf16"])
INF = float("inf")


def _heads():
    from volume_integration import heads
    return heads


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


# ---- candidates of long rows ----
NOTE = 96       # bytes that sample_labels notes a row in its scratch: a double, two floats, the state, 16 counts, padding
KEPT = 512      # candidates a warp keeps


def _candidates(z, u, **settings):
    """(labels, [M, W] counts, [M, W, KEPT] places) of a call with a scratch of the test's own."""
    lib, p = ha.load(), ctypes.c_void_p
    lib.vi_sample_labels_scratch_bytes.argtypes = [ctypes.c_int, ctypes.POINTER(ha.Matrix), ctypes.POINTER(Sampling)]
    lib.vi_sample_labels_scratch_bytes.restype = ctypes.c_uint64
    lib.vi_sample_labels.argtypes = [ctypes.c_int, ctypes.POINTER(ha.Matrix), p, ctypes.POINTER(Sampling), p, p,
                                     ctypes.c_uint64, p]
    M = z.shape[0]
    warps = 16 if M <= torch.cuda.get_device_properties(0).multi_processor_count else 8
    s = Sampling(**{**dict(temperature=1.0, top_p=1.0, min_p=0.0, top_k=0), **settings})
    n = lib.vi_sample_labels_scratch_bytes(ha.DTYPE[z.dtype], ha.matrix(z), ctypes.byref(s))
    lists = warps * KEPT * 4
    assert n >= M * (NOTE + lists)
    scratch = torch.zeros(n, device="cuda", dtype=torch.uint8)
    label = torch.empty(M, device="cuda", dtype=torch.int64)
    assert lib.vi_sample_labels(ha.DTYPE[z.dtype], ha.matrix(z), p(u.data_ptr()), ctypes.byref(s), p(label.data_ptr()),
                                p(scratch.data_ptr()), n, p(torch.cuda.current_stream().cuda_stream)) == 0, lib.vi_last_error()
    notes = scratch[:M * NOTE].view(torch.int32).reshape(M, NOTE // 4)
    assert int(notes[:, 4].min()) >= 0 and int(notes[:, 4].max()) <= 2  # the state: the layout is the one read here
    return label, notes[:, 5:5 + warps], scratch[M * NOTE:M * (NOTE + lists)].view(torch.int32).reshape(M, warps, KEPT)


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,V,order", [(200, 9000, "image"), (200, 9001, "rows"), (3, 50257, "rows"), (3, 50257, "image")])
def test_candidates_of_long_rows_are_labels_of_the_row(M, V, order, dt):
    # the last warp's part of these rows holds fewer labels than it keeps candidates; a floor under a peak, clipped and flat
    # logits put the sample's tail into one value, so that no guess leaves anything out
    g = _gen(V)
    u = torch.rand(M, generator=g, device="cuda")
    peak = torch.zeros(M, V, device="cuda")
    peak[:, 5] = 9.0
    clipped = torch.randn(M, V, generator=g, device="cuda").clamp(-0.5, 0.5) * 40
    masked = torch.randn(M, V, generator=g, device="cuda")
    masked[:, 100:] = -INF
    kinds = [peak, clipped, torch.full((M, V), 0.25, device="cuda"), masked]
    for kind in kinds:
        z = kind.t().contiguous().t() if order == "image" else kind
        z = z.to(dt) if order == "image" else z.to(dt).contiguous()
        assert (z.stride(0) == 1) == (order == "image")
        first = torch.zeros(M, device="cuda", dtype=torch.int64)
        if order == "rows":  # places are counted from the 16 bytes' boundary in front of a row
            first = (z.data_ptr() + torch.arange(M, device="cuda") * z.stride(0) * z.element_size()) % 16 // z.element_size()
        for settings in (dict(top_p=0.9), dict(top_p=0.999, temperature=1.9), dict(top_k=V - 1), dict(top_k=50),
                         dict(min_p=1e-30), dict(min_p=0.5), dict(temperature=0.0), dict(min_p=1e-30, temperature=1e4)):
            label, counts, places = _candidates(z, u, **settings)
            kept = torch.arange(KEPT, device="cuda") < counts[:, :, None]
            low, high = first[:, None, None], first[:, None, None] + V
            outside = kept & ((places < low) | (places >= high))
            assert not bool(outside.any()), (settings, int(outside.sum()))
            assert int(counts.sum(1).max()) <= V, settings
            assert torch.equal(label[:3].cpu(), dl.sample(z[:3], u[:3], **settings)), settings


# ---- logits far from zero ----
def _u_at_borders(z, t, p, g):
    """For each row a u just behind the start of a kept label's share, by the definition with top-p alone."""
    z = z.double().cpu()
    us = []
    for row in z:
        w = torch.exp((row - row.max()) / t)
        order = torch.sort(row, descending=True, stable=True).indices
        before = w[order].cumsum(0) - w[order]
        n = max(1, int((before < p * w.sum()).sum()))
        kept = torch.sort(order[:n]).values
        run = w[kept].cumsum(0)
        at = int(torch.randint(n // 2, n, (1,), generator=g))
        us.append(torch.tensor(float((run[at] - w[kept[at]]) / run[-1]) + 2e-7).float())
    return torch.stack(us).cuda()


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("shift,t", [(30.0, 0.1), (100.0, 0.5), (1000.0, 1.0), (1000.0, 0.1), (-1000.0, 0.1), (8000.0, 0.5)])
def test_top_p_of_long_rows_far_from_zero(shift, t, dt):
    # in float32 thousands of labels are kept, each about 1e-4 of the mass: a mass that is off by more than the kernel allows
    # for keeps another number of them, and every border moves
    g, cpu = _gen(int(shift) % 97), torch.Generator().manual_seed(int(shift) % 89)
    M, V, p = 100, 9000, 0.7
    step = {F32: 0.0, F16: 2.0 ** -10, BF16: 2.0 ** -7}[dt] * abs(shift)  # spread over some of the type's steps
    z = (shift + max(t, step) * torch.randn(M, V, generator=g, device="cuda")).to(dt)
    u = _u_at_borders(z, t, p, cpu)
    got = _heads().sample_labels(z, u, temperature=t, top_p=p)
    want = dl.sample(z, u, temperature=t, top_p=p)
    assert torch.equal(got.cpu(), want), int((got.cpu() != want).sum())


# ---- settings at the ends of their ranges ----
@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("V,order", [(20, "rows"), (40, "image"), (400, "image"), (3000, "rows"), (9000, "rows"), (9000, "image")])
def test_settings_by_row_outside_their_ranges(V, order, dt):
    # a min_p above 1 keeps the largest, as 1 does; top_p and min_p that are no numbers, and a negative min_p, are off
    nan = float("nan")
    g = _gen(V)
    M = 48
    z = hl.matrix(M, V, dt, g, order, scale=3.0)
    z[7, [3, V - 1]] = z[7].max() + 1  # two largest
    u = torch.rand(M, generator=g, device="cuda")
    m = torch.tensor([1.0, 1.5, 2.0, 1e30, INF, nan, -1.0, 7.0, 0.0, 0.3, -INF, 1 + 2.0 ** -23], device="cuda").repeat(4)
    p = torch.tensor([nan, 0.9, 1.5, INF, nan, 0.0, -1.0, -INF], device="cuda").repeat(6)
    means = m.nan_to_num(nan=0.0, posinf=1.0).clamp(0, 1)
    for extra in (dict(), dict(temperature=0.5), dict(top_k=9), dict(top_p=0.8)):
        got = _heads().sample_labels(z, u, min_p=m, **extra)
        assert torch.equal(got.cpu(), dl.sample(z, u, min_p=means, **extra)), extra
    got = _heads().sample_labels(z, u, top_p=p, min_p=0.01)
    assert torch.equal(got.cpu(), dl.sample(z, u, top_p=p.nan_to_num(nan=1.0), min_p=0.01))


# ---- waits that run out ----
def test_a_wait_that_runs_out_for_one_lane_ends_the_block(monkeypatch):
    # every copy arrives, but one lane's wait counts as run out: its warp, or block, gives up as one, and the status word says so
    heads, g = _heads(), _gen(43)
    w = heads.quantize_rows(hl.matrix(64, 64, F32, g))
    u = torch.rand(70000, generator=g, device="cuda")
    calls = []
    for dt in (F16, BF16):
        for order in ("rows", "image"):
            x = hl.matrix(70000, 64, dt, g, order)
            calls.append(lambda x=x: heads.linear_act_int8(x, w, residual=x, activation="gelu"))
    for dt in (F32, F16, BF16):
        z = hl.matrix(70000, 21, dt, g, "image")
        calls.append(lambda z=z: heads.sample_labels(z, u, min_p=0.02))
    before = [call() for call in calls]
    assert heads.device_status() == 0
    monkeypatch.setenv("VI_HEADS_TEST_TIMEOUT", "2")
    for call in calls:
        call()
        assert heads.device_status(reset=True) == 8
    monkeypatch.delenv("VI_HEADS_TEST_TIMEOUT")
    for call, want in zip(calls, before):
        assert torch.equal(call(), want)
    assert heads.device_status() == 0


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,V,order", [(3000, 400, "image"), (3001, 1000, "image"), (3000, 33, "image"), (300, 500, "rows")])
def test_min_p_of_1_draws_among_the_largest(M, V, order, dt):
    g = _gen(V)
    z = hl.matrix(M, V, dt, g, order, scale=3.0)
    top = z.amax(1)
    z[::3, V // 2] = top[::3]                                     # two largest
    z[1::3, 7] = torch.nextafter(top[1::3].float(), top[1::3].float() - 1).to(dt)  # float32: the next one below
    u = torch.rand(M, generator=g, device="cuda")
    for t, m in ((1.0, 1.0), (3.0, 1.0), (1.0, 1 - 2.0 ** -24), (1.0, 1 - 2e-7), (0.5, 1 - 1e-6), (1.0, 1 - 1e-5), (1.0, 1 - 4e-5)):
        got = _heads().sample_labels(z, u, temperature=t, min_p=m)
        assert torch.equal(got.cpu(), dl.sample(z, u, temperature=t, min_p=m)), (t, m)


@pytest.mark.parametrize("dt", **TYPES)
def test_min_p_of_1_takes_no_longer_than_less(dt):
    # an image of 257 to 1024 labels: its largest logits, whose weight is 1, are no cause for doing a pixel again in 64 bits
    # (10 to 17 times as long)
    heads, g = _heads(), _gen(44)
    z = hl.matrix(100000, 400, dt, g, "image", scale=3.0)
    u = torch.rand(100000, generator=g, device="cuda")

    def fastest(min_p):
        times = []
        for _ in range(8):
            ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            ends[0].record()
            heads.sample_labels(z, u, min_p=min_p)
            ends[1].record()
            torch.cuda.synchronize()
            times.append(ends[0].elapsed_time(ends[1]))
        return min(times)

    usual = fastest(0.5)
    assert fastest(1.0) <= 3 * usual and fastest(1 - 1e-5) <= 3 * usual


# ---- launches ----
@pytest.mark.parametrize("M,K,launches", [(4, 5000, 3), (4, 4000, 2), (9, 5000, 3), (9, 48, 3)])
def test_linear_act_int8_copies_unaligned_weights_once(M, K, launches):
    # weights whose rows do not lie 16 bytes apart are copied by one launch; beside it: up to 8 rows of up to 4096 features are
    # one, else the rows' quantising and the product
    heads, g, lib = _heads(), _gen(K), ha.load()
    lib.vi_kernel_launches.restype = ctypes.c_uint64
    x = hl.matrix(M, K, BF16, g)
    q, s = heads.quantize_rows(hl.matrix(70, K, F32, g))
    odd = torch.empty(70, K + 1, device="cuda", dtype=torch.int8)[:, :K]
    odd.copy_(q)
    before = lib.vi_kernel_launches()
    y = heads.linear_act_int8(x, (odd, s))
    assert lib.vi_kernel_launches() - before == launches
    assert torch.equal(y, heads.linear_act_int8(x, (q, s)))


def test_quantize_rows_of_images_from_several_threads():
    # calls of a C host's threads that need different amounts of shared memory, at once
    import threading
    lib, p, g = ha.load(), ctypes.c_void_p, _gen(47)
    lib.vi_quantize_rows.argtypes = [ctypes.c_int, ctypes.POINTER(ha.Matrix), ctypes.POINTER(ha.Matrix), p, p]
    sizes, out, failed = (2600, 1000, 2600, 1200), [], []
    for K in sizes:
        x = hl.matrix(100, K, BF16, g, "image")
        out.append((x, torch.zeros(100, (K + 15) // 16 * 16, device="cuda", dtype=torch.int8)[:, :K], torch.zeros(100, device="cuda")))
    torch.cuda.synchronize()

    def calls(x, q, scale):
        for _ in range(3000):
            if lib.vi_quantize_rows(2, ha.matrix(x), ha.matrix(q), p(scale.data_ptr()), None):
                failed.append(lib.vi_last_error())

    threads = [threading.Thread(target=calls, args=o) for o in out]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, (len(failed), failed[0])
    for x, q, scale in out:
        wq, ws = dl.quantize(x)
        assert torch.equal(q, wq) and torch.equal(scale, ws)


# ---- scales ----
@pytest.mark.parametrize("power", [-140, -96, -95, -80, -1, 0, 126, 127])
def test_scales_are_the_rounded_quotients_of_every_significand(power):
    x = torch.arange(1 << 23, 1 << 24, dtype=torch.int64).double().mul(2.0 ** -23).mul(2.0 ** power)
    x = x[x <= torch.finfo(F32).max].float()  # under 2^-126 some are rounded: still values of the type
    # rounded twice, which is as once: no quotient by 127 lies within 1 / 254 of a step of float32's halves but on them
    want = (x.double() / 127).float()
    _, scale = _heads().quantize_rows(x.cuda().unsqueeze(1))
    assert torch.equal(scale.cpu(), want)


# ---- draws at the ends of u ----
@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("M,V,order", [(40, 21, "rows"), (300, 100, "image"), (300, 300, "image"), (40, 3000, "rows"),
                                       (40, 20000, "rows"), (200, 50001, "rows"), (40, 20000, "image")])
def test_u_of_0_draws_the_first_label_with_weight(M, V, order, dt):
    # however little it weighs beside the ones behind it
    g = _gen(V)
    z = hl.matrix(M, V, dt, g, order, scale=30.0)
    z[::2, :V // 3] = -INF
    u = torch.zeros(M, device="cuda")
    for t in (1.0, 0.7, 3.0):
        w = torch.exp((z.double() - z.double().amax(1, keepdim=True)) / t)
        want = (w > 2.0 ** -999).to(torch.uint8).argmax(1)  # the kernel's least weight is 2^-1000
        for settings in (dict(), dict(top_p=1.0), dict(min_p=0.0, top_k=2 * V)):
            got = _heads().sample_labels(z, u, temperature=t, **settings)
            assert torch.equal(got, want), (t, settings, int((got != want).sum()))


@pytest.mark.parametrize("dt", **TYPES)
@pytest.mark.parametrize("V,order", [(20, "rows"), (40, "image"), (400, "image"), (3000, "rows"), (9000, "rows"), (9000, "image")])
def test_infinite_logits_take_all_mass_at_any_temperature(V, order, dt):
    g = _gen(V)
    M = 64
    z = hl.matrix(M, V, dt, g, order, scale=3.0)
    where = torch.randint(1, V, (M, 2), generator=g, device="cuda")
    z.scatter_(1, where, INF)
    u = torch.rand(M, generator=g, device="cuda")
    u[:2], u[2] = 0.0, 1 - 2.0 ** -24
    first, second = where.amin(1), where.amax(1)
    want = torch.where((u < 0.5) | (first == second), first, second)
    for t in (0.5, 1e6, 1e35, INF, torch.full((M,), INF, device="cuda")):
        for settings in (dict(), dict(top_k=5), dict(top_p=0.999), dict(min_p=0.2), dict(top_k=V - 1, top_p=1.0)):
            got = _heads().sample_labels(z, u, temperature=t, **settings)
            assert torch.equal(got, want), (t if isinstance(t, float) else "rows", settings, int((got != want).sum()))
