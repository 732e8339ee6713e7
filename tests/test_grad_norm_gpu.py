"""Global gradient norm and clipping against 64-bit values.

Bounds: a vector's squares are summed in 32 bits with at most 8 roundings (8 x 2^-24 of a sum of squares, half of that of
its root), everything above in 64: norm within 2^-21 of itself. The factor max_norm / (norm + 1e-6) takes three
roundings more, the product one, and the result is rounded to its type (eps / 2)."""
import pytest
import torch

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def tensors_of(sizes, dtype, seed=0, scale=1.0, offset=0):
    """Views of one flat buffer, `offset` elements into it: starts of every alignment."""
    g = torch.Generator().manual_seed(seed)
    flat = (torch.randn(sum(sizes) + offset, generator=g) * scale).to(dtype).cuda()
    return flat, list(flat[offset:].split(sizes))


def wide_norm(ts):
    return torch.sqrt(sum((t.double() ** 2).sum() for t in ts))


def check(ts, max_norm, norm=None):
    from evox_b200.grad_kernels import clip_grad_norm_

    before = [t.double() for t in ts]
    want = wide_norm(before)
    got = clip_grad_norm_(ts, max_norm)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - float(want)) <= 2.0**-21 * float(want) + 1e-45
    f = min(1.0, max_norm / (float(want) + 1e-6))
    for t, b in zip(ts, before):
        if f == 1.0:
            assert torch.equal(t.double(), b)
            continue
        tiny = 2.0**-25 if t.dtype == torch.float16 else 2.0**-149 if t.dtype == torch.float32 else 2.0**-134
        tol = (b * f).abs() * (torch.finfo(t.dtype).eps / 2 * 1.01 + 2.0**-20) + tiny
        assert bool(((t.double() - b * f).abs() <= tol).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [[1], [0, 1, 0], [3, 5, 7, 1, 2], [4096], [4095, 4097, 1], [65536, 256] * 3, [1000003], [17] * 95, [17] * 96, [31] * 97,
                                   [5, 0, 1025] * 167, [1] * 1499, [1] * 1500, [3] * 1501, [7] * 3300])
def test_norm_and_clip(cuda, sizes, dtype):
    from evox_b200.grad_kernels import grad_norm

    for offset in (0, 1, 3):
        flat, ts = tensors_of(sizes, dtype, offset=offset)
        want = float(wide_norm(ts))
        keep = flat.clone()
        assert abs(float(grad_norm(ts)) - want) <= 2.0**-21 * want
        assert torch.equal(flat, keep)
        check(ts, 0.25 * want + 1e-3)
        assert torch.equal(flat[:offset], keep[:offset])
        check(ts, 1e6)


@gpu
def test_large_and_mixed(cuda):
    g = torch.Generator(device="cuda").manual_seed(0)
    ts = [torch.randn(30_000_001, generator=g, device=cuda), torch.randn(4097, 1023, generator=g, device=cuda).bfloat16(),
          torch.randn(9, 9, 9, generator=g, device=cuda).half(), torch.randn((), generator=g, device=cuda)]
    check(ts, 3.0)


@gpu
def test_more_elements_than_32_bits_count(cuda):
    n = 2**31 + 77
    flat = torch.empty(n + 1, dtype=torch.bfloat16, device=cuda).normal_(generator=torch.Generator(device="cuda").manual_seed(0))
    from evox_b200.grad_kernels import clip_grad_norm_

    tail = flat[-100:].double()
    head = flat[:100].double()
    want = float(torch.sqrt(sum(c.float().square().sum(dtype=torch.float64) for c in flat[1:].split(2**27))))
    norm = float(clip_grad_norm_(flat[1:], 1.0))
    assert abs(norm - want) <= 2.0**-20 * want
    f = 1.0 / (norm + 1e-6)
    assert bool(((flat[-100:].double() - tail * f).abs() <= (tail * f).abs() * 2.0**-7.9 + 1e-40).all())
    assert bool(((flat[1:100].double() - head[1:] * f).abs() <= (head[1:] * f).abs() * 2.0**-7.9 + 1e-40).all()) and float(flat[0]) == float(head[0])


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e-15, 1e15, 1e22, 3e30])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_squares_outside_the_range_of_32_bits(cuda, dtype, scale):
    from evox_b200.grad_kernels import grad_norm

    _, ts = tensors_of([1000, 3], dtype, scale=scale)
    want = float(wide_norm(ts))
    assert abs(float(grad_norm(ts)) - want) <= 2.0**-21 * want
    if scale > 1:
        check(ts, 1.0)


@gpu
def test_values_that_are_not_finite(cuda):
    from evox_b200.grad_kernels import clip_grad_norm_

    for bad, first, rest in ((float("inf"), float("nan"), 0.0), (float("nan"), float("nan"), float("nan"))):
        ts = [torch.ones(100, device=cuda), torch.ones(50, device=cuda)]
        ts[1][7] = bad
        norm = clip_grad_norm_(ts, 1.0)
        twin = [torch.ones(100, device=cuda), torch.ones(50, device=cuda)]
        twin[1][7] = bad
        for p, q in zip(twin, ts):  # what torch's own rule gives
            f = torch.clamp(1.0 / (torch.tensor(bad, device=cuda).abs() + 1e-6), max=1.0)
            assert torch.equal(torch.nan_to_num(p * f, nan=-7.0), torch.nan_to_num(q, nan=-7.0))
        assert not torch.isfinite(norm)
    zeros = [torch.zeros(10, device=cuda), torch.zeros(0, device=cuda)]
    assert float(clip_grad_norm_(zeros, 1.0)) == 0.0 and not zeros[0].any()
    ones = [torch.ones(64, device=cuda)]
    assert float(clip_grad_norm_(ones, 0.0)) == 8.0 and not ones[0].any()


@gpu
def test_repeats_streams_graphs_and_versions(cuda):
    from evox_b200.grad_kernels import clip_grad_norm_, grad_norm

    sizes = [100003, 17, 0, 65536, 5]
    flat, ts = tensors_of(sizes, torch.float32, offset=1)
    start = flat.clone()
    version = ts[0]._version
    norm = clip_grad_norm_(ts, 1.0).clone()
    assert ts[0]._version > version
    want = flat.clone()
    side = torch.cuda.Stream()
    flat.copy_(start)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = clip_grad_norm_(ts, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(flat, want) and torch.equal(norm, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = clip_grad_norm_(ts, 1.0)
    for _ in range(2):
        flat.copy_(start)
        graph.replay()
        assert torch.equal(flat, want) and torch.equal(norm, captured)
    flat.copy_(start)
    assert torch.equal(grad_norm(ts), norm) and torch.equal(grad_norm(ts[0]), grad_norm([ts[0]]))


@gpu
def test_shared_memory_is_refused(cuda):
    from evox_b200._cabi import EvoxKernelError
    from evox_b200.grad_kernels import clip_grad_norm_, grad_norm

    x = torch.ones(100, device=cuda)
    for ts in ([x, x], [x[:60], x[50:]], [x[50:], x[:60]], [x, torch.ones(3, device=cuda), x[99:]]):
        with pytest.raises(EvoxKernelError, match="share memory"):
            clip_grad_norm_(ts, 1.0)
    assert abs(float(grad_norm([x, x])) - 200**0.5) <= 2.0**-20 * 15  # reading twice is well defined
    with pytest.raises(EvoxKernelError, match="contiguous"):
        grad_norm([torch.ones(4, 4, device=cuda).t()[:2]])
    with pytest.raises(EvoxKernelError, match="one CUDA device"):
        grad_norm([x, torch.ones(3)])
    assert bool((x == 1).all())


def test_refusals():
    from evox_b200._cabi import EvoxKernelError
    from evox_b200.grad_kernels import clip_grad_norm_, grad_norm

    for fn in (grad_norm, lambda t: clip_grad_norm_(t, 1.0)):
        with pytest.raises(EvoxKernelError, match="empty"):
            fn([])
        with pytest.raises(EvoxKernelError, match="CUDA device"):
            fn([torch.zeros(3)])
        with pytest.raises(EvoxKernelError, match="float64"):
            fn([torch.zeros(3, dtype=torch.float64)])
    for bad in (-1.0, float("nan")):
        with pytest.raises(EvoxKernelError, match="max_norm"):
            clip_grad_norm_([torch.zeros(3)], bad)


def test_c_entry_refuses_bad_arguments():
    from ctypes import c_int32, c_int64, c_uint64

    from evox_b200 import _cabi

    lib = _cabi.lib

    def call(address=(256, 4096), numel=(4, 4), dtype=(2, 2), n=2, max_norm=1.0, clip=1, norm=256, ws=256, nbytes=1 << 20):
        return lib.evox_clip_grad_norm((c_uint64 * len(address))(*address), (c_int64 * len(numel))(*numel), (c_int32 * len(dtype))(*dtype), n, max_norm,
                                       clip, norm, ws, nbytes, None)

    for kw in (dict(norm=None), dict(ws=None), dict(ws=257), dict(n=-1), dict(dtype=(2, 3)), dict(numel=(4, -1)), dict(numel=(4, 1 << 41)),
               dict(address=(256, 0)), dict(address=(256, 4098)), dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(address=(256, 268)),
               dict(address=(268, 256))):
        assert call(**kw) == -1, kw
        assert b"clip_grad_norm" in lib.evox_last_error()
    assert call(nbytes=8) == -3
