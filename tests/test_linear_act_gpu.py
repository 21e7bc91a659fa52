"""Products with bias, activation and residual in their epilogue against the same in float64: types, sizes no tile divides, rows that are
apart, every form of the tensor cores' product, places that must stay as they were, streams and captured graphs."""
import pytest
import torch

from iian_b200.ops.cuda_backend import CudaKernels, KernelError
from scored_model import ACTIVATIONS

pytestmark = pytest.mark.gpu
K = CudaKernels
BF, F32 = torch.bfloat16, torch.float32
SLOPE = {"none": 1.0, "silu": 1.1, "gelu": 1.13, "gelu_tanh": 1.13, "relu": 1.0}


def reference(x, w, bias, act, residual):
    y = x.double() @ w.double().t()
    if bias is not None:
        y = y + bias.double()
    a = ACTIVATIONS[act](y)
    return y, a if residual is None else a + residual.double()


def tolerance(x, w, y, ref, act, out_dtype, tc):
    """Elementwise, from the arithmetic.  The float32 chain of the general kernel rounds once a product (2^-24 of the partial sum, K times);
    the tensor cores' adds 16 products at a time and cuts off (2^-23 of the partial sum and of the largest product, each of K / 16 + 1
    times), a partial sum being at most sum |x w|.  Joining parts, bias and residual are roundings of 2^-24 of what is added: 32 of them are
    allowed for.  The activation stretches all that by its steepest slope and is itself off by a few units in the last place
    and, gelu, by 3e-7 |y| / 2; then the rounding into out, half a step."""
    total = x.double().abs() @ w.double().abs().t()
    k = x.shape[1]
    chain = total * ((2 * (k / 16 + 1)) * 2.0 ** -23 if tc else k * 2.0 ** -24) + 32 * 2.0 ** -24 * (total + y.abs() + ref.abs())
    slope = SLOPE.get(act, 0.0) if act != "relu2" else 2 * y.abs() + chain
    return slope * chain + (1e-6 + 2.0 ** -22) * y.abs() + 2e-6 * ref.abs() + torch.finfo(out_dtype).eps / 2 * ref.abs() + 1e-30


def check(n, k, m, dtype=BF, out_dtype=BF, act="none", bias=True, residual=False, form=0, seed=0, wdtype=None, rdtype=F32):
    g = torch.Generator("cuda").manual_seed(seed + n + k + m)
    x = torch.randn(n, k, device="cuda", generator=g).to(dtype)
    w = (torch.randn(m, k, device="cuda", generator=g) * 0.05).to(wdtype or dtype)
    b = torch.randn(m, device="cuda", generator=g) if bias else None
    r = (torch.randn(n, m, device="cuda", generator=g) * 2).to(rdtype) if residual else None
    out = torch.full((n, m), float("nan"), device="cuda", dtype=out_dtype)
    K().linear_act(x, w, out, bias=b, activation=act, residual=r, form=form)
    y, ref = reference(x, w, b, act, r)
    tc = dtype == BF and w.dtype == BF and k % 8 == 0
    assert ((out.double() - ref).abs() <= tolerance(x, w, y, ref, act, out_dtype, tc)).all()
    K().check_device_status()


SIZES = [(1, 64, 32), (1, 8, 1), (1, 4096, 130), (3, 1000, 64), (17, 72, 50), (64, 2048, 257), (127, 136, 100), (128, 512, 128), (129, 512, 128), (255, 264, 1416),
         (256, 64, 256), (257, 1024, 520), (600, 320, 777), (1100, 2048, 1024)]


@pytest.mark.parametrize("n,k,m", SIZES)
@pytest.mark.parametrize("act,bias,residual,out_dtype", [("gelu", True, False, BF), ("none", False, True, F32), ("silu", True, True, F32)])
def test_bfloat16(n, k, m, act, bias, residual, out_dtype):
    check(n, k, m, BF, out_dtype, act, bias, residual)


@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("dtype,out_dtype", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("n", [5, 200])
def test_activations(act, dtype, out_dtype, n):
    check(n, 160, 224, dtype, out_dtype, act, True, True, rdtype=BF if out_dtype == BF else F32)


@pytest.mark.parametrize("n,k,m", [(1, 1, 1), (1, 70, 50), (4, 4096, 64), (16, 128, 6200), (17, 33, 31), (61, 1024, 520), (301, 1024, 333), (301, 70, 65), (700, 256, 1024)])
def test_float32(n, k, m):
    check(n, k, m, F32, F32, "gelu_tanh", True, True)
    check(n, k, m, F32, F32, "none", False, False)


@pytest.mark.parametrize("n,k,m", [(1, 4097, 130), (3, 1001, 64), (8, 77, 6150), (9, 258, 4100), (16, 31, 100), (16, 514, 6144), (17, 1023, 65), (84, 3199, 181),
                                   (301, 515, 1030), (1025, 130, 2050)])
def test_float32_rows_that_do_not_begin_on_16_bytes(n, k, m):
    check(n, k, m, F32, F32, "silu", True, True)
    check(n, k, m, F32, F32, "none", False, False)
    wide = torch.randn(n, 4 * k + 3, device="cuda")                  # 4 k floats wide: every piece of a row but its place is whole
    x, w, out = wide[:, 1:1 + 4 * k], torch.randn(m, 4 * k, device="cuda") * 0.05, torch.empty(n, m, device="cuda")
    K().linear_act(x, w, out)
    y, ref = reference(x, w, None, "none", None)
    assert ((out.double() - ref).abs() <= tolerance(x, w, y, ref, "none", F32, False)).all()


@pytest.mark.parametrize("tile", range(5))
@pytest.mark.parametrize("groups", [1, 2, 3, 4, 6, 8])
def test_every_form_of_float32(tile, groups):
    if tile > 2 and groups % 2:
        pytest.skip("eight warps")
    for n, k, m in ((1, 1, 1), (3, 40, 33), (33, 1027, 65), (70, 516, 130), (9, 4096, 64)):
        check(n, k, m, F32, F32, "gelu", True, True, form=tile + 1 | groups << 8)


@pytest.mark.parametrize("bad", [6 | 1 << 8, 255 | 1 << 8, 1 << 8, 1, 1 | 9 << 8, 4 | 1 << 8, -1])
def test_forms_that_float32_has_not(bad):
    x, w, out = (torch.zeros(s, device="cuda") for s in ((4, 64), (8, 64), (4, 8)))
    with pytest.raises(KernelError):
        K().linear_act(x, w, out, form=bad)


@pytest.mark.parametrize("k,m", [(64, 32), (700, 4100), (1027, 65), (1024, 2048), (2049, 1030), (4096, 500)])
def test_float32_rows_have_the_same_bits_in_any_batch(k, m):
    x, w, b = torch.randn(1100, k, device="cuda"), torch.randn(m, k, device="cuda") * 0.05, torch.randn(m, device="cuda")
    whole = torch.empty(1100, m, device="cuda")
    K().linear_act(x, w, whole, bias=b, activation="silu")
    for first, n in ((0, 1), (5, 7), (12, 17), (40, 61), (100, 301), (450, 650)):
        wide = torch.empty(n, k + 1, device="cuda")
        wide[:, 1:] = x[first: first + n]
        for rows in (x[first: first + n], wide[:, 1:]):
            out = torch.empty(n, m, device="cuda")
            K().linear_act(rows, w, out, bias=b, activation="silu")
            assert torch.equal(out, whole[first: first + n])


def test_float32_rows_far_apart():
    store = torch.empty(8 * 2 ** 28 + 64, device="cuda")             # the ninth row begins 8 GB on
    x = store.as_strided((9, 64), (2 ** 28, 1))
    x.copy_(torch.randn(9, 64, device="cuda"))
    w, out = torch.randn(70, 64, device="cuda") * 0.05, torch.empty(9, 70, device="cuda")
    K().linear_act(x, w, out)
    y, ref = reference(x, w, None, "none", None)
    assert ((out.double() - ref).abs() <= tolerance(x, w, y, ref, "none", F32, False)).all()


@pytest.mark.parametrize("n,k,m", [(1, 4096, 155), (40, 1027, 300)])
def test_float32_captured_and_on_another_stream(n, k, m):
    x, w, b = torch.randn(n, k, device="cuda"), torch.randn(m, k, device="cuda") * 0.05, torch.randn(m, device="cuda")
    out, r = torch.empty(n, m, device="cuda"), torch.randn(n, m, device="cuda")
    want = torch.empty(n, m, device="cuda")
    K().linear_act(x, w, want, bias=b, activation="gelu", residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K().linear_act(x, w, out, bias=b, activation="gelu", residual=r)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K().linear_act(x, w, out, bias=b, activation="gelu", residual=r)
        K().linear_act(x, w, r, residual=r)
    x.mul_(0.5)
    start = r.clone()
    K().linear_act(x, w, want, bias=b, activation="gelu", residual=start)
    second = start.clone()
    K().linear_act(x, w, second, residual=second)
    graph.replay()
    assert torch.equal(out, want) and torch.equal(r, second)


@pytest.mark.parametrize("n,k,m", [(2, 64, 40), (33, 1027, 70)])
def test_float32_infinities_and_nan_stay_in_their_rows(n, k, m):
    x, w = torch.randn(n, k, device="cuda"), torch.randn(m, k, device="cuda")
    clean, out = torch.empty(n, m, device="cuda"), torch.empty(n, m, device="cuda")
    K().linear_act(x, w, clean)
    x[n - 1, k - 1], w[m - 1, 0] = float("nan"), float("inf")
    K().linear_act(x, w, out)
    assert torch.equal(out[: n - 1, : m - 1], clean[: n - 1, : m - 1])
    assert out[n - 1].isnan().all() and not out[: n - 1, m - 1].isfinite().any()


@pytest.mark.parametrize("dtype,wdtype,k", [(BF, F32, 64), (F32, BF, 64), (BF, BF, 71), (BF, BF, 4)])
def test_what_the_tensor_cores_do_not_take(dtype, wdtype, k):
    check(33, k, 50, dtype, BF, "relu", True, True, wdtype=wdtype)


def form(pair, bn, ks):
    return int(pair) | bn << 1 | ks << 16


@pytest.mark.parametrize("n", [1, 31, 128, 130, 300])
@pytest.mark.parametrize("pair,bn,ks", [(0, 32, 1), (0, 48, 3), (0, 112, 6), (0, 176, 5), (0, 240, 2), (0, 256, 8), (0, 256, 1), (1, 32, 1), (1, 64, 4), (1, 96, 3),
                                        (1, 224, 2), (1, 256, 4), (1, 256, 1)])
def test_every_form(n, pair, bn, ks):
    check(n, 1048, 700, BF, F32, "relu", True, True, form(pair, bn, ks))          # (no width of a tile divides 700)
    check(n, 1048, 701, BF, BF, "silu", True, False, form(pair, bn, ks))          # entries, not groups of four


@pytest.mark.parametrize("n", [1, 16, 61, 100, 128])
@pytest.mark.parametrize("bn,ks", [(32, 1), (48, 8), (64, 2), (96, 3), (112, 6), (128, 1), (128, 4)])
def test_every_form_of_few_rows(n, bn, ks):
    check(n, 1048, 700, BF, F32, "relu", True, True, form(0, bn, ks) | 1 << 14)
    check(n, 1048, 701, BF, BF, "silu", True, False, form(0, bn, ks) | 1 << 14)
    check(n, 72, 36, BF, F32, "none", True, True, form(0, bn, min(ks, 2)) | 1 << 14)


@pytest.mark.parametrize("n,bn", [(4, 144), (129, 64)])
def test_few_rows_are_few(n, bn):
    x, w, out = (torch.zeros(s, device="cuda", dtype=BF) for s in ((n, 1024), (64, 1024), (n, 64)))
    with pytest.raises(KernelError):
        K().linear_act(x, w, out, form=form(0, bn, 1) | 1 << 14)


@pytest.mark.parametrize("bad", [(0, 16, 1), (0, 40, 1), (0, 272, 1), (1, 48, 1), (0, 64, 9), (1, 64, 5), (0, 64, 0), (0, 32, 8 + 1)])
def test_forms_there_are_none_of(bad):
    x, w, out = (torch.zeros(s, device="cuda", dtype=BF) for s in ((4, 1024), (64, 1024), (4, 64)))
    with pytest.raises(KernelError):
        K().linear_act(x, w, out, form=form(*bad))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,k,m", [(3, 64, 40), (150, 128, 72), (20, 70, 33)])
def test_rows_apart_and_what_lies_between_them(dtype, n, k, m):
    g = torch.Generator("cuda").manual_seed(n)
    wide_x = torch.randn(n + 2, k + 24, device="cuda", generator=g).to(dtype)
    wide_r = torch.randn(n + 2, m + 8, device="cuda", generator=g)
    wide_o = torch.full((n + 2, m + 12), 7.0, device="cuda", dtype=F32)
    x, r, out = wide_x[:n, 8:8 + k], wide_r[:n, 4:4 + m], wide_o[:n, 4:4 + m]
    w = (torch.randn(m, k, device="cuda", generator=g) * 0.05).to(dtype)
    K().linear_act(x, w, out, activation="gelu", residual=r)
    y, ref = reference(x, w, None, "gelu", r)
    assert ((out.double() - ref).abs() <= tolerance(x, w, y, ref, "gelu", F32, dtype == BF and k % 8 == 0)).all()
    untouched = wide_o.clone()
    untouched[:n, 4:4 + m] = 7.0
    assert (untouched == 7.0).all()
    x = wide_x[:n, 4:4 + k]                                         # rows that do not begin on 16 bytes
    K().linear_act(x, w, out, activation="gelu", residual=r)
    y, ref = reference(x, w, None, "gelu", r)
    assert ((out.double() - ref).abs() <= tolerance(x, w, y, ref, "gelu", F32, False)).all()
    one = wide_r[:1, 4:4 + m].expand(n, m)                         # one row for all of them
    K().linear_act(x, w, out, activation="gelu", residual=one)
    y, ref = reference(x, w, None, "gelu", one)
    assert ((out.double() - ref).abs() <= tolerance(x, w, y, ref, "gelu", F32, dtype == BF and k % 8 == 0)).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,k,m", [(1, 256, 64), (60, 3000, 192), (400, 512, 300)])
def test_into_the_residual_itself(dtype, n, k, m):
    g = torch.Generator("cuda").manual_seed(n)
    x = torch.randn(n, k, device="cuda", generator=g).to(dtype)
    w = (torch.randn(m, k, device="cuda", generator=g) * 0.05).to(dtype)
    b = torch.randn(m, device="cuda", generator=g)
    stream = torch.randn(n, m, device="cuda", generator=g)
    other = torch.empty_like(stream)
    K().linear_act(x, w, other, bias=b, residual=stream)
    K().linear_act(x, w, stream, bias=b, residual=stream)
    assert torch.equal(stream, other)


@pytest.mark.parametrize("n", [1, 70, 300])
def test_same_bits_again(n):
    g = torch.Generator("cuda").manual_seed(n)
    x = torch.randn(n, 2048, device="cuda", generator=g).to(BF)
    w = (torch.randn(640, 2048, device="cuda", generator=g) * 0.05).to(BF)
    outs = [torch.empty(n, 640, device="cuda") for _ in range(3)]
    for o in outs:
        K().linear_act(x, w, o, activation="silu")
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_nothing_to_do_and_special_values():
    z = lambda *s, t=BF: torch.zeros(*s, device="cuda", dtype=t)      # noqa: E731
    K().linear_act(z(0, 64), z(32, 64), z(0, 32))
    K().linear_act(z(5, 64), z(0, 64), z(5, 0))
    for dtype in (BF, F32):
        x = torch.ones(3, 64, device="cuda", dtype=dtype)
        x[1, 5] = float("inf")
        x[2, 7] = float("nan")
        w = torch.ones(40, 64, device="cuda", dtype=dtype)
        out = z(3, 40, t=F32)
        for act in ("none", "relu", "relu2", "silu", "gelu", "gelu_tanh"):
            K().linear_act(x, w, out, activation=act)
            assert torch.isfinite(out[0]).all() and (out[1] == float("inf")).all() and torch.isnan(out[2]).all(), act
        K().linear_act(-x, w, out, activation="silu")                  # far below 0: what an overflowing exponential must not make of it
        assert (out[0].abs() <= 64 * 2.0 ** -80).all()


def test_refusals():
    k, z = K(), lambda *s, t=BF: torch.zeros(*s, device="cuda", dtype=t)      # noqa: E731
    x, w, out = z(4, 64), z(32, 64), z(4, 32)
    with pytest.raises(KernelError, match="tanh"):
        k.linear_act(x, w, out, activation="tanh")
    for kw in ({"bias": z(31, t=F32)}, {"bias": z(32)}, {"residual": z(3, 32)}, {"residual": z(4, 32, t=torch.float16)}, {"bias": torch.zeros(32)},
               {"residual": torch.zeros(4, 32)}):
        with pytest.raises(KernelError):
            k.linear_act(x, w, out, **kw)
    with pytest.raises(KernelError):
        k.linear_act(x, w, z(4, 33))
    with pytest.raises(KernelError):
        k.linear_act(x, w, z(4, 32, t=torch.float16))
    with pytest.raises(KernelError, match="contiguous rows"):
        k.linear_act(z(64, 4).t(), w, out)
    with pytest.raises(KernelError, match="overlap"):
        k.linear_act(z(1, 64).expand(4, 64), w, out)
    with pytest.raises(KernelError, match="overlap"):
        k.linear_act(x, w, z(1, 32).expand(4, 32))
    with pytest.raises(KernelError):
        k.linear_act(x, z(64, 64)[:, :32].t(), out)
    both = z(4, 64, t=F32)
    with pytest.raises(KernelError, match="place of out"):
        k.linear_act(x, w, both[:, :32], residual=both.view(8, 32)[:4])
    with pytest.raises(KernelError, match="place of out"):
        k.linear_act(x, w, both[:, :32].view(BF)[:, :32], residual=both[:, :32])


def test_two_streams_at_once():
    g = torch.Generator("cuda").manual_seed(3)
    n, k, m = 90, 4096, 1024
    sets = [((torch.randn(n, k, device="cuda", generator=g)).to(BF), (torch.randn(m, k, device="cuda", generator=g) * 0.05).to(BF),
             torch.empty(n, m, device="cuda")) for _ in range(2)]
    want = []
    for x, w, o in sets:
        K().linear_act(x, w, o, activation="gelu")
        want.append(o.clone())
        o.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(20):
        for s, (x, w, o) in zip(streams, sets):
            with torch.cuda.stream(s):
                K().linear_act(x, w, o, activation="gelu")
    torch.cuda.synchronize()
    assert all(torch.equal(o, v) for (_, _, o), v in zip(sets, want))
    K().check_device_status()


@pytest.mark.parametrize("dtype,n", [(BF, 1), (BF, 40), (BF, 300), (F32, 20)])
def test_captured_and_replayed(dtype, n):
    g = torch.Generator("cuda").manual_seed(n)
    k, m = 512, 384
    x = torch.randn(n, k, device="cuda", generator=g).to(dtype)
    up = (torch.randn(m, k, device="cuda", generator=g) * 0.05).to(dtype)
    down = (torch.randn(k, m, device="cuda", generator=g) * 0.05).to(dtype)
    act, stream = torch.empty(n, m, device="cuda", dtype=dtype), torch.zeros(n, k, device="cuda")

    def run():
        K().linear_act(x, up, act, activation="gelu")
        K().linear_act(act, down, stream, residual=stream)

    run()                                                             # (compiles and sets attributes)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in (1, 2):
        x.copy_(torch.randn(n, k, device="cuda", generator=g))
        stream.normal_(0.0, 1.0, generator=g)
        start = stream.clone()
        graph.replay()
        replayed = stream.clone()
        stream.copy_(start)
        run()
        assert torch.equal(replayed, stream)
