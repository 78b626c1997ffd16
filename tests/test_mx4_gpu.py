"""Microscaled 4-bit kernels against their definition in 64 bits, with bounds derived from the roundings (tests/helpers/mx4_oracle.py)."""

import pytest
import torch

from parallax_b200 import ops
from tests.helpers import mx4_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _status():
    yield
    if torch.cuda.is_available():
        from parallax_b200.ops import cuda as cu

        cu.check_status(torch.device("cuda", torch.cuda.current_device()))


def _matrix(rows, K, seed, lo=117, hi=126):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 256, (rows, K // 2), generator=g, dtype=torch.uint8),
            torch.randint(lo, hi, (rows, K // 32), generator=g, dtype=torch.uint8))


def _normal(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


# ------------------------------------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 96), (77, 1056), (1000, 4096)])
def test_quantisation(rows, K, dtype):
    x = _normal(rows, K, seed=rows, dtype=torch.float32)
    x = (x * torch.exp(4 * _normal(rows, 1, seed=1, dtype=torch.float32))).to(dtype)
    want = ops.reference.quant_mx4_rows(x)
    codes, scales = ops.quant_mx4_rows(x.to(DEV))
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
    assert torch.equal(ops.expand_mx4_rows(codes, scales).cpu().double(), oracle.values(*want))


def test_quantisation_on_borders_and_extremes():
    b = (oracle.MAGS[1:] + oracle.MAGS[:-1]).float() / 2
    b = torch.cat([b, oracle.MAGS.float()])
    v = torch.cat([b, torch.nextafter(b, torch.tensor(float("inf"))), torch.nextafter(b, torch.tensor(-float("inf")))])
    v = torch.cat([v, -v])
    v = torch.nn.functional.pad(v[v.abs() <= 6], (0, 31 * 4))[:31 * 3].view(3, 31)
    rows = [torch.cat([r, torch.tensor([6.0])]) * 2.0 ** p for r in v for p in (-126, -30, 0, 17, 120)]
    rows += [torch.full((32,), m) for m in (3.0, 3.0000002, 6.0, 6.0000005, 1.5, 5.9999995, 2.0 ** -149, 2.0 ** -127, 3e38, -0.0, 0.0)]
    for bad in (float("nan"), float("inf"), -float("inf")):
        r = torch.randn(32)
        r[7] = bad
        rows.append(r)
    x = torch.stack(rows)
    codes, scales = ops.quant_mx4_rows(x.to(DEV))
    want = ops.reference.quant_mx4_rows(x)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
    got, ref = ops.expand_mx4_rows(codes, scales).cpu(), ops.reference.expand_mx4_rows(*want)
    assert torch.equal(torch.nan_to_num(got, nan=-1.25), torch.nan_to_num(ref, nan=-1.25))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantisation_of_strided_and_unaligned_rows(dtype):
    base = _normal(9, 300, dtype=dtype).to(DEV)
    for x in (base[:1, 5:37].expand(7, 32), base[:, 8:104], base[:, 1:97], base[1:, 3:35], base[:, :96].t().contiguous().t(), base[:, ::2][:, :96]):
        want = ops.reference.quant_mx4_rows(x.cpu())
        got = ops.quant_mx4_rows(x)
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_every_code_and_scale():
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)[:, :16 * 16].contiguous()
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16).contiguous()
    want = ops.reference.expand_mx4_rows(codes, scales)
    got = ops.expand_mx4_rows(*_dev(codes, scales)).cpu()
    assert torch.equal(torch.nan_to_num(got, nan=-1.25), torch.nan_to_num(want, nan=-1.25))
    buf = torch.zeros(1 + codes.numel(), dtype=torch.uint8, device=DEV)      # codes that start on an odd byte
    odd = buf[1:].view_as(codes)
    odd.copy_(codes)
    got = ops.expand_mx4_rows(odd, scales.to(DEV)).cpu()
    assert torch.equal(torch.nan_to_num(got, nan=-1.25), torch.nan_to_num(want, nan=-1.25))


def test_no_rows():
    codes, scales = ops.quant_mx4_rows(torch.zeros(0, 64, device=DEV))
    assert codes.shape == (0, 32) and scales.shape == (0, 2) and ops.expand_mx4_rows(codes, scales).shape == (0, 64)
    w = _dev(*_matrix(64, 64, 0))
    assert ops.linear_mx4(torch.zeros(0, 64, device=DEV).bfloat16(), ops.Mx4Weight.pack(*w)).shape == (0, 64)
    assert ops.linear_mx4_rows(codes, scales, *w).shape == (0, 64)


@pytest.mark.parametrize("experts,N,K", [(1, 1, 32), (1, 130, 160), (3, 128, 128), (2, 300, 96), (5, 257, 1056)])
def test_layout(experts, N, K):
    codes, scales = _matrix(experts * N, K, N, 0, 129)
    for _ in range(2):
        want = ops.Mx4Weight.pack(codes, scales, experts=experts)
        got = ops.Mx4Weight.pack(*_dev(codes, scales), experts=experts)
        assert torch.equal(got.data.cpu(), want.data)
        assert torch.equal(torch.nan_to_num(got.row_scale.cpu(), nan=-1.0), torch.nan_to_num(want.row_scale, nan=-1.0))
        g = torch.Generator().manual_seed(N)                # and scales of all sizes, NaN among them
        scales = torch.randint(0, 256, scales.shape, generator=g, dtype=torch.uint8)
    view = torch.zeros(codes.shape[0], codes.shape[1] + 3, dtype=torch.uint8, device=DEV)
    view[:, 3:] = codes.to(DEV)
    assert torch.equal(ops.Mx4Weight.pack(view[:, 3:], scales.to(DEV), experts=experts).data.cpu(), want.data)


# ------------------------------------------------------------------------------------------------ products
def _product_case(T, N, K, bias=False, residual=False, act="", seed=0, lo=117, hi=126):
    x, (codes, scales) = _normal(T, K, seed=seed), _matrix(N, K, seed + 1, lo, hi)
    n_out = N // 2 if act else N
    b, r = (_normal(N, seed=seed + 2) if bias else None), (_normal(T, n_out, seed=seed + 3) if residual else None)
    return x, codes, scales, b, r


EPIS = {"": ops.EPI_NONE, "silu": ops.EPI_SILU_MUL, "clip": ops.EPI_CLIP_GLU}
SIZES = [(1, 1, 32), (1, 128, 128), (2, 130, 160), (7, 64, 4096), (8, 384, 1056), (9, 1000, 96), (16, 257, 2880), (17, 128, 512), (32, 640, 352),
         (33, 257, 992), (64, 512, 1536), (65, 300, 128), (100, 777, 2048), (128, 256, 736), (129, 384, 4096), (200, 1300, 320), (256, 129, 1024),
         (257, 640, 608), (515, 259, 1312), (1100, 515, 288)]


@pytest.mark.parametrize("T,N,K", SIZES)
def test_product(T, N, K):
    x, codes, scales, b, r = _product_case(T, N, K, True, True, seed=T)
    w, wide = ops.Mx4Weight.pack(*_dev(codes, scales)), oracle.values(codes, scales)
    for bias, res in ((None, None), (b, None), (b, r)):
        got = ops.linear_mx4(x.to(DEV), w, *_dev(bias, res))
        oracle.within(got, *oracle.linear(x.double(), wide, bias, res), (T, N, K, bias is None, res is None))


@pytest.mark.parametrize("act", ["silu", "clip"])
@pytest.mark.parametrize("T,N,K", [(1, 128, 32), (1, 1280, 2880), (5, 256, 4096), (31, 384, 160), (120, 640, 1024), (300, 256, 2080)])
def test_gated_product(T, N, K, act):
    x, codes, scales, b, _ = _product_case(T, N, K, True, act=act, seed=T + 40)
    w, wide = ops.Mx4Weight.pack(*_dev(codes, scales)), oracle.values(codes, scales)
    for bias in (None, b):
        got = ops.linear_mx4(x.to(DEV), w, *_dev(bias), epi=EPIS[act], limit=1.5)
        oracle.within(got, *oracle.linear(x.double(), wide, bias, None, act, 1.5), (T, N, K, bias is None))


@pytest.mark.parametrize("T", [1, 6, 40, 300])
def test_scales_of_all_sizes(T):
    """Powers from the smallest up, some beyond 128 (rows with factors), rows with a NaN scale, rows of x with an infinity."""
    N, K = 260, 320
    x, codes, scales, *_ = _product_case(T, N, K, seed=3)
    scales = torch.randint(0, 100, scales.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(1))
    scales[7], scales[8] = 141, torch.randint(120, 150, (10,), dtype=torch.uint8)
    scales[9, 4] = 255
    scales[200, 9] = 254
    scales[200, :9] = 250
    w = ops.Mx4Weight.pack(*_dev(codes, scales))
    want, bound = oracle.linear(x.double(), oracle.values(codes, scales))
    got = ops.linear_mx4(x.to(DEV), w).cpu()
    small = torch.ones(N, dtype=torch.bool)
    small[200] = False
    tiny = 2.0 ** -133                        # (results below the subnormals of bf16)
    oracle.within(got[:, small], want[:, small], bound[:, small] + tiny)
    big = want[:, 200].abs() > 3.5e38        # a row whose values pass the largest bf16 number
    assert torch.isinf(got[:, 200][big]).all() and torch.isnan(got[:, 9]).all()
    x[0, 5] = float("inf")
    got = ops.linear_mx4(x.to(DEV), w).cpu()[0]
    assert not torch.isfinite(got[:8]).any()


@pytest.mark.parametrize("T", [3, 70, 260])
def test_strides_and_unaligned_operands(T):
    N, K = 261, 192
    x, codes, scales, b, r = _product_case(T, N, K, True, True, seed=T)
    w, want = ops.Mx4Weight.pack(*_dev(codes, scales)), oracle.linear(x.double(), oracle.values(codes, scales), b, r)
    wide = torch.full((T, 600), 7.0, dtype=torch.bfloat16, device=DEV)
    for at in (8, 3):                                   # on 16 bytes, and not
        wide[:, at:at + K] = x.to(DEV)
        oracle.within(ops.linear_mx4(wide[:, at:at + K], w, *_dev(b, r)), *want, at)
    oracle.within(ops.linear_mx4(x.to(DEV).t().contiguous().t(), w, *_dev(b, r)), *want, "columns first")
    for at in (8, 5):
        dst = torch.full((T, 500), 7.0, dtype=torch.bfloat16, device=DEV)
        res = torch.zeros((T, 700), dtype=torch.bfloat16, device=DEV)
        res[:, at + 1:at + 1 + N] = r.to(DEV)
        bias = torch.cat([b[:1], b]).to(DEV)[1:]
        out = dst[:, at:at + N]
        assert ops.linear_mx4(x.to(DEV), w, bias, res[:, at + 1:at + 1 + N], out=out) is out
        oracle.within(out, *want, at)
        assert bool((dst[:, :at] == 7).all()) and bool((dst[:, at + N:] == 7).all())
    one = x[:1].expand(T, K)                            # rows that are one and the same, and a residual that is
    want = oracle.linear(one.double(), oracle.values(codes, scales), b, r[:1].expand(T, N))
    oracle.within(ops.linear_mx4(x[:1].to(DEV).expand(T, K), w, b.to(DEV), r[:1].to(DEV).expand(T, N)), *want, "expanded")
    with pytest.raises(ops.KernelError):
        ops.linear_mx4(x.to(DEV), w, out=torch.zeros(1, N, dtype=torch.bfloat16, device=DEV).expand(T, N))
    want = oracle.linear(x.double(), oracle.values(codes, scales), b, r)
    acc = r.to(DEV)                                     # the residual is written in place
    oracle.within(ops.linear_mx4(x.to(DEV), w, b.to(DEV), acc, out=acc), *want, "in place")


@pytest.mark.parametrize("T,N,K,act", [(203, 5120, 25600, ""), (256, 5120, 8192, ""), (230, 2560, 12800, "silu"), (13, 25600, 5120, "silu"),
                                       (60, 25600, 5120, ""), (90, 12800, 5120, ""), (1000, 5120, 5120, ""), (8192, 12288, 4096, "silu")])
def test_large_products_again_and_again(T, N, K, act):
    """Every SM loads at full rate, so that loads end in any order: the same bits every time, and samples against 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(T)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8, device=DEV)
    scales = torch.randint(112, 120, (N, K // 32), generator=g, dtype=torch.uint8, device=DEV)
    x = torch.randn(T, K, generator=g, device=DEV).bfloat16()
    w = ops.Mx4Weight.pack(codes, scales)
    first = ops.linear_mx4(x, w, epi=EPIS[act])
    for _ in range(10):
        assert torch.equal(ops.linear_mx4(x, w, epi=EPIS[act]), first)
    tokens = torch.randperm(T)[:32]
    rows = torch.arange(N).view(-1, 128)[torch.randperm(N // 128)[:2]].flatten()       # two blocks of weight rows
    want = oracle.linear(x.cpu()[tokens].double(), oracle.values(codes.cpu()[rows], scales.cpu()[rows]), act=act)
    cols = rows if not act else (rows.view(-1, 128)[:, :1] // 2 + torch.arange(64)).flatten()
    oracle.within(first.cpu()[tokens][:, cols], *want)


# ------------------------------------------------------------------------------------------------ both operands in 4 bits
@pytest.mark.parametrize("T,N,K", SIZES)
def test_product_of_codes(T, N, K):
    x, codes, scales, b, r = _product_case(T, N, K, True, True, seed=T + 9)
    xc, xs = ops.reference.quant_mx4_rows(x)
    a, wide = oracle.values(xc, xs), oracle.values(codes, scales)
    d = _dev(xc, xs, codes, scales)
    for bias, res in ((None, None), (b, None), (b, r)):
        got = ops.linear_mx4_rows(*d, *_dev(bias, res))
        oracle.within(got, *oracle.linear(a, wide, bias, res), (T, N, K, bias is None, res is None))


@pytest.mark.parametrize("T", [2, 40, 300])
def test_product_of_codes_with_every_scale(T):
    """Scales of either side from end to end, as far as their products stay within fp32, and NaN."""
    N, K = 140, 288
    g = torch.Generator().manual_seed(T)
    xc, xs = _matrix(T, K, 1, 0, 1)
    codes, scales = _matrix(N, K, 2, 0, 1)
    xs = torch.randint(100, 160, xs.shape, dtype=torch.uint8, generator=g)
    scales = torch.randint(100, 160, scales.shape, dtype=torch.uint8, generator=g)
    xs[0], scales[3], scales[4] = 250, 5, 2
    scales[5, 2], xs[1, 8] = 255, 255
    a, wide = oracle.values(xc, xs), oracle.values(codes, scales)
    want, bound = oracle.linear(a, wide)
    got = ops.linear_mx4_rows(*_dev(xc, xs, codes, scales)).cpu()
    # row 0 (2^123) times scales up to 2^32 passes 2^128, the end of fp32: partial sums of both signs are infinite there, and what is
    # left of them is any of NaN and the infinities. Where the sum of the magnitudes stays below, so does every partial sum.
    held = ~(a.abs() @ wide.abs().t() > 2.0 ** 127)
    oracle.within(got[held], want[held], bound[held])
    assert not torch.isfinite(got[~held & (want.abs() > 2.0 ** 128)]).any()


# ------------------------------------------------------------------------------------------------ experts
def _experts_case(T, E, k, K, I, seed=0, biases=True):
    g = torch.Generator().manual_seed(seed)
    x, base = _normal(T, K, seed=seed), _normal(T, K, seed=seed + 1)
    (c1, s1), (c2, s2) = _matrix(E * 2 * I, K, seed + 2), _matrix(E * K, I, seed + 3)
    b1, b2 = (_normal(E * 2 * I, seed=seed + 4), _normal(E * K, seed=seed + 5)) if biases else (None, None)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).int()
    return x, base, c1, s1, c2, s2, b1, b2, ids, torch.rand(T, k, generator=g)


@pytest.mark.parametrize("clip", [False, True])
@pytest.mark.parametrize("T,E,k,K,I", [(1, 8, 2, 64, 64), (1, 32, 4, 2880, 192), (5, 4, 4, 352, 128), (40, 16, 4, 512, 320), (130, 3, 2, 160, 64),
                                       (700, 6, 3, 288, 192)])
def test_experts(T, E, k, K, I, clip):
    x, base, c1, s1, c2, s2, b1, b2, ids, wts = _experts_case(T, E, k, K, I, seed=T, biases=clip)
    if T > 4:
        ids[1, 0] = ids[1, 1]                   # an expert twice in a row
        ids[2] = -1                             # none
        ids[3, 0] = E
        ids[4:, 0] = 1                          # and one with many rows
    w1, w2 = ops.Mx4Weight.pack(*_dev(c1, s1), experts=E), ops.Mx4Weight.pack(*_dev(c2, s2), experts=E)
    for bs in (base, None):
        want = oracle.experts(x, ids, wts, oracle.values(c1, s1).view(E, 2 * I, K), oracle.values(c2, s2).view(E, K, I), bs, clip, 1.5,
                              None if b1 is None else b1.view(E, -1), None if b2 is None else b2.view(E, -1))
        got = ops.moe_ffn_mx4(*_dev(x, ids, wts), w1, w2, base=None if bs is None else bs.to(DEV), act_mode=int(clip), limit=1.5,
                              b1=None if b1 is None else b1.to(DEV), b2=None if b2 is None else b2.to(DEV))
        oracle.within(got, *want, (T, E, bs is None))


@pytest.mark.parametrize("T,E,k,K,I", [(1, 5, 1, 32, 64), (2, 8, 4, 2880, 192), (3, 4, 5, 352, 320), (8, 6, 2, 4096, 64), (1, 3, 16, 160, 1024)])
def test_experts_of_a_few_pairs(T, E, k, K, I):
    """Every pair on its own: experts twice in a row, none, and NaN weights and scales of experts that are not asked."""
    x, base, c1, s1, c2, s2, b1, b2, _ids, wts = _experts_case(T, E, min(k, E), K, I, seed=T + 50)
    g = torch.Generator().manual_seed(k)
    ids, wts = torch.randint(0, E - 1, (T, k), generator=g).int(), torch.rand(T, k, generator=g)
    ids[0, 0], wts[0, 0] = (E if k > 1 else 0), (float("nan") if k > 1 else 0.5)
    ids[-1, -1] = -1 if k > 1 or T > 1 else 0
    s1.view(E, -1)[E - 1], s2.view(E, -1)[E - 1] = 255, 255
    w1, w2 = ops.Mx4Weight.pack(*_dev(c1, s1), experts=E), ops.Mx4Weight.pack(*_dev(c2, s2), experts=E)
    want = oracle.experts(x, ids, wts, oracle.values(c1, s1).view(E, 2 * I, K), oracle.values(c2, s2).view(E, K, I), base, True, 1.5,
                          b1.view(E, -1), b2.view(E, -1))
    from parallax_b200.ops import _lib

    assert _lib.lib().pxl_moe_mx4_few_takes(T, k, K, I) == 1
    got = ops.moe_ffn_mx4(*_dev(x, ids, wts), w1, w2, base=base.to(DEV), act_mode=1, limit=1.5, b1=b1.to(DEV), b2=b2.to(DEV))
    oracle.within(got, *want)


@pytest.mark.parametrize("T", [35, 60, 80, 111, 144, 201, 260, 330, 440, 700])
def test_experts_of_every_tile_height(T):
    """Rows per expert from a few to two tiles' worth, evenly over the experts and nearly all on one."""
    E, k, K, I = 4, 2, 1056, 192
    x, base, c1, s1, c2, s2, _b1, _b2, ids, wts = _experts_case(T, E, k, K, I, seed=T, biases=False)
    w1, w2 = ops.Mx4Weight.pack(*_dev(c1, s1), experts=E), ops.Mx4Weight.pack(*_dev(c2, s2), experts=E)
    v1, v2 = oracle.values(c1, s1).view(E, 2 * I, K), oracle.values(c2, s2).view(E, K, I)
    skewed = ids.clone()
    skewed[3:, 0], skewed[3:, 1] = 2, 2
    for which in (ids, skewed):
        want = oracle.experts(x, which, wts, v1, v2, base, False, 1.5, None, None)
        for _ in range(3):
            oracle.within(ops.moe_ffn_mx4(*_dev(x, which, wts), w1, w2, base=base.to(DEV)), *want)


def test_experts_too_wide_for_shared_memory():
    """Few pairs, but more columns of the inner rows than the direct form holds: the sorted form takes them."""
    from parallax_b200.ops import _lib

    T, E, k, K, I = 1, 2, 2, 32, 401408
    assert _lib.lib().pxl_moe_mx4_few_takes(T, k, K, I) == 0
    x, base, c1, s1, c2, s2, _b1, _b2, ids, wts = _experts_case(T, E, k, K, I, seed=3, biases=False)
    w1, w2 = ops.Mx4Weight.pack(*_dev(c1, s1), experts=E), ops.Mx4Weight.pack(*_dev(c2, s2), experts=E)
    want = oracle.experts(x, ids, wts, oracle.values(c1, s1).view(E, 2 * I, K), oracle.values(c2, s2).view(E, K, I), base, False, 1.5, None, None)
    oracle.within(ops.moe_ffn_mx4(*_dev(x, ids, wts), w1, w2, base=base.to(DEV)), *want)


@pytest.mark.parametrize("T,N,K", [(700, 5120, 12288), (1500, 5120, 12800), (2048, 20480, 6144), (4000, 2047, 8192)])
def test_wide_tiles_of_deep_products(T, N, K):
    """Tiles of more than 192 rows, one and several per CTA, with a residual; samples against 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(N)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8, device=DEV)
    scales = torch.randint(112, 120, (N, K // 32), generator=g, dtype=torch.uint8, device=DEV)
    x, r = torch.randn(T, K, generator=g, device=DEV).bfloat16(), torch.randn(T, N, generator=g, device=DEV).bfloat16()
    xc, xs = ops.quant_mx4_rows(x)
    got, got44 = ops.linear_mx4(x, ops.Mx4Weight.pack(codes, scales), residual=r), ops.linear_mx4_rows(xc, xs, codes, scales, residual=r)
    tokens, rows = torch.cat([torch.randperm(T)[:32], torch.tensor([0, 255, 256, T - 1])]), torch.randperm(N)[:300]
    w, res = oracle.values(codes.cpu()[rows], scales.cpu()[rows]), r.cpu()[tokens][:, rows]
    oracle.within(got.cpu()[tokens][:, rows], *oracle.linear(x.cpu()[tokens].double(), w, residual=res))
    oracle.within(got44.cpu()[tokens][:, rows], *oracle.linear(oracle.values(xc.cpu()[tokens], xs.cpu()[tokens]), w, residual=res))


# ------------------------------------------------------------------------------------------------ streams, graphs, repeats
def _layer(x, w_in, w_out, wr, ids, wts, w1, w2):
    """The operators one behind the other, as a layer uses them."""
    h = ops.linear_mx4(x, w_in, epi=ops.EPI_SILU_MUL)
    h = ops.linear_mx4(h, w_out, residual=x)
    h = ops.linear_mx4_rows(*ops.quant_mx4_rows(h), *wr, residual=h)
    return ops.moe_ffn_mx4(h, ids, wts, w1, w2, base=h)


def _layer_inputs(T, seed=0):
    K, I, E = 256, 384, 6
    w_in, w_out = ops.Mx4Weight.pack(*_dev(*_matrix(2 * I, K, 1))), ops.Mx4Weight.pack(*_dev(*_matrix(K, I, 2)))
    w1 = ops.Mx4Weight.pack(*_dev(*_matrix(E * 2 * I, K, 3)), experts=E)
    w2 = ops.Mx4Weight.pack(*_dev(*_matrix(E * K, I, 4)), experts=E)
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:2] for _ in range(T)]).int()
    return [*_dev(_normal(T, K, seed=seed)), w_in, w_out, _dev(*_matrix(K, K, 5)), *_dev(ids, torch.rand(T, 2, generator=g)), w1, w2]


@pytest.mark.parametrize("T", [1, 37, 300])
def test_layer_on_another_stream_in_a_chain_and_in_graphs(T):
    from parallax_b200.ops import cuda as cu

    a, b = _layer_inputs(T, 0), _layer_inputs(T, 1)
    want_a, want_b = _layer(*a), _layer(*b)
    assert torch.equal(want_a, _layer(*a))                      # the same sums in the same order
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = {}
    for _ in range(4):                                          # two calls at once
        for name, s, args in (("a", s1, a), ("b", s2, b)):
            with torch.cuda.stream(s):
                outs[name] = _layer(*args)
    torch.cuda.synchronize()
    assert torch.equal(outs["a"], want_a) and torch.equal(outs["b"], want_b)
    with cu.launch_chain():
        got = _layer(*a)
    assert torch.equal(got, want_a)
    graphs = []
    for args in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _layer(*args)
        graphs.append((g, out))
    for _ in range(3):
        for s, (g, _out) in zip((s1, s2), graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want_a) and torch.equal(graphs[1][1], want_b)


@pytest.mark.parametrize("T,N,K", [(300, 40000, 64), (1000, 20000, 32), (20, 60000, 96), (60, 40000, 224), (2, 60000, 64)])
def test_many_short_tiles_in_a_chain(T, N, K):
    """Weights are read ahead of a kernel's turn, here more blocks of them than its first tile has."""
    from parallax_b200.ops import cuda as cu

    x, r = _normal(T, K, seed=1).to(DEV), _normal(T, N, seed=2).to(DEV)
    codes, scales = _dev(*_matrix(N, K, 3))
    w, xq = ops.Mx4Weight.pack(codes, scales), ops.quant_mx4_rows(x)
    want, want44 = ops.linear_mx4(x, w, residual=r), ops.linear_mx4_rows(*xq, codes, scales, residual=r)
    torch.cuda.synchronize()
    with cu.launch_chain():
        got = [ops.linear_mx4(x, w, residual=r) for _ in range(3)]
        got44 = [ops.linear_mx4_rows(*xq, codes, scales, residual=r) for _ in range(3)]
    assert all(torch.equal(y, want) for y in got) and all(torch.equal(y, want44) for y in got44)
    oracle.within(want, *oracle.linear(x.cpu().double(), oracle.values(codes.cpu(), scales.cpu()), residual=r.cpu()))


@pytest.mark.parametrize("T", [1, 40, 300])
def test_weights_made_inside_a_chain(T):
    from parallax_b200.ops import cuda as cu

    x, weight = _normal(T, 512, seed=1).to(DEV), _normal(640, 512, seed=2).to(DEV)
    q = ops.quant_mx4_rows(weight)
    want = ops.linear_mx4(x, ops.Mx4Weight.pack(*q)), ops.linear_mx4_rows(*ops.quant_mx4_rows(x), *q), ops.linear(x, ops.expand_mx4_rows(*q))
    torch.cuda.synchronize()
    with cu.launch_chain():
        rows = ops.quant_mx4_rows(x)
        got = ops.linear_mx4_rows(*rows, *ops.quant_mx4_rows(weight))
        assert torch.equal(got, want[1])
    for _ in range(3):
        with cu.launch_chain():
            q = ops.quant_mx4_rows(weight)
            a = ops.linear_mx4(x, ops.Mx4Weight.pack(*q))
            c = ops.linear(x, ops.expand_mx4_rows(*q))
        assert torch.equal(a, want[0]) and torch.equal(c, want[2])


def test_refusals():
    x = torch.zeros(2, 64, device=DEV)
    w = ops.Mx4Weight.pack(*_dev(*_matrix(64, 64, 0)))
    for call in (lambda: ops.linear_mx4(x, w), lambda: ops.quant_mx4_rows(x[:, :48]), lambda: ops.quant_mx4_rows(x.half()),
                 lambda: ops.linear_mx4(x.bfloat16(), w, bias=torch.zeros(64).bfloat16()),
                 lambda: ops.linear_mx4(x.bfloat16(), ops.Mx4Weight.pack(*_matrix(64, 64, 0)))):
        with pytest.raises(ops.KernelError):
            call()


# ------------------------------------------------------------------------------------------------ engine
@pytest.mark.parametrize("clipped", [False, True])
def test_engine_with_packed_experts(clipped):
    """Requests through the serving engine, and its experts' layers against the definition."""
    from parallax_b200.engine.engine import Engine
    from parallax_b200.engine.request import SamplingParams
    from parallax_b200.models.config import config_from_hf

    sizes = dict(hidden_size=512, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2, head_dim=64, vocab_size=1024,
                 num_experts_per_tok=4, max_position_embeddings=2048, rope_theta=10000.0)
    if clipped:
        cfg = config_from_hf(dict(architectures=["GptOssForCausalLM"], model_type="gpt_oss", intermediate_size=320, moe_intermediate_size=320,
                                  num_local_experts=8, sliding_window=32, attention_bias=True,
                                  layer_types=["sliding_attention", "full_attention"], **sizes))
    else:
        cfg = config_from_hf(dict(architectures=["Qwen3MoeForCausalLM"], model_type="qwen3_moe", intermediate_size=512,
                                  moe_intermediate_size=192, num_experts=16, norm_topk_prob=True, **sizes))
    plain = Engine(cfg, device=DEV + ":0", num_blocks=64, max_batch_size=4)
    eng = Engine(cfg, device=DEV + ":0", num_blocks=64, max_batch_size=4, expert_format="mxfp4")
    outs = eng.generate([list(range(5, 60)), [7, 8, 9]], SamplingParams(max_new_tokens=6, temperature=0.0, ignore_eos=True))
    assert all(len(o) == 6 for o in outs)
    assert eng.stages[0].model.weight_bytes() < plain.stages[0].model.weight_bytes()
    for T in (1, 3, 50):
        x = _normal(T, cfg.hidden_size, seed=T)
        for lw in eng.stages[0].model.layers:
            moe = lw.moe
            ids, wts = moe.route(x.to(DEV))
            E, w1, w2 = cfg.num_experts, moe.mx4["w1"], moe.mx4["w2"]
            wide = [oracle.values(*(t.cpu() for t in w.unpack())).view(E, w.rows, w.cols) for w in (w1, w2)]
            b = [None if t is None else t.cpu().view(E, -1) for t in (moe.b1, moe.b2)]
            want = oracle.experts(x, ids.cpu(), wts.cpu(), *wide, x, clipped, moe.limit, *b)
            oracle.within(moe.forward(x.to(DEV), x.to(DEV)), *want, T)
