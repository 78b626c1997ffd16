"""Calls of the microscaled 4-bit operators that their other tests leave out: operands on odd addresses, the forms of a few pairs of tokens
and experts that split K over a cluster, and the same bits on every run."""

import pytest
import torch

from parallax_b200 import ops
from parallax_b200.ops import _lib, cuda as cu
from tests.helpers import mx4_oracle as oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _status():
    yield
    if torch.cuda.is_available():
        cu.check_status(torch.device("cuda", torch.cuda.current_device()))


def _matrix(rows, K, seed, lo=117, hi=126):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 256, (rows, K // 2), generator=g, dtype=torch.uint8),
            torch.randint(lo, hi, (rows, K // 32), generator=g, dtype=torch.uint8))


def _normal(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).bfloat16()


def _experts(T, E, k, K, I, seed=0, missing=False):
    """Inputs of moe_ffn_mx4 on the GPU, and what its definition gives with a base. `missing`: the first pair's expert does not exist."""
    g = torch.Generator().manual_seed(seed)
    (c1, s1), (c2, s2) = _matrix(E * 2 * I, K, seed + 2), _matrix(E * K, I, seed + 3)
    x, base, b1, b2 = _normal(T, K, seed=seed), _normal(T, K, seed=seed + 1), _normal(E * 2 * I, seed=seed + 4), _normal(E * K, seed=seed + 5)
    ids, wts = torch.randint(0, E, (T, k), generator=g).int(), torch.rand(T, k, generator=g)
    if missing:
        ids[0, 0] = -1
    want = oracle.experts(x, ids, wts, oracle.values(c1, s1).view(E, 2 * I, K), oracle.values(c2, s2).view(E, K, I), base, True, 1.5,
                          b1.view(E, -1), b2.view(E, -1))
    w1, w2 = (ops.Mx4Weight.pack(c.to(DEV), s.to(DEV), experts=E) for c, s in ((c1, s1), (c2, s2)))
    return dict(x=x.to(DEV), ids=ids.to(DEV), weights=wts.to(DEV), w1=w1, w2=w2, base=base.to(DEV), act_mode=1, limit=1.5, b1=b1.to(DEV),
                b2=b2.to(DEV)), want


def _at(t, offset):
    """The same values `offset` elements behind the start of an allocation."""
    return torch.cat([t.new_zeros(offset), t.flatten()])[offset:].view(t.shape)


@pytest.mark.parametrize("offset", [1, 4])
@pytest.mark.parametrize("T,few", [(2, 1), (90, 0)])
def test_experts_with_operands_on_odd_addresses(T, few, offset):
    E, k, K, I = 4, 2, 352, 128
    args, want = _experts(T, E, k, K, I, seed=T)
    assert _lib.lib().pxl_moe_mx4_few_takes(T, k, K, I) == few
    args |= {n: _at(args[n], offset) for n in ("x", "base", "b1", "b2", "ids", "weights")}
    oracle.within(ops.moe_ffn_mx4(**args), *want)


@pytest.mark.parametrize("offset", [1, 4])
def test_bf16_experts_with_operands_on_odd_addresses(offset):
    T, E, k, K, I = 33, 4, 2, 128, 64
    g = torch.Generator().manual_seed(0)
    x, base, w1, w2 = (t.to(DEV) for t in (_normal(T, K), _normal(T, K, seed=1), _normal(E * 2 * I, K, seed=2), _normal(E * K, I, seed=3)))
    ids, wts = torch.randint(0, E, (T, k), generator=g).int().to(DEV), torch.rand(T, k, generator=g).to(DEV)
    want = ops.moe_ffn(x, ids, wts, w1, w2, E, base=base)
    assert torch.equal(ops.moe_ffn(_at(x, offset), ids, wts, w1, w2, E, base=_at(base, offset)), want)
    wide = torch.zeros(T, 3 * K, dtype=torch.bfloat16, device=DEV)
    wide[:, K:2 * K], wide[:, 2 * K:] = x, base
    assert torch.equal(ops.moe_ffn(wide[:, K:2 * K], ids, wts, w1, w2, E, base=wide[:, 2 * K:]), want)


@pytest.mark.parametrize("missing", [False, True])
@pytest.mark.parametrize("T,E,k,K,I", [(1, 3, 16, 640, 4096), (1, 20, 13, 96, 5056), (1, 2, 1, 65536, 64), (2, 3, 2, 57376, 64)])
def test_experts_of_a_few_pairs_over_a_cluster(T, E, k, K, I, missing):
    """More columns than a CTA holds of a row: of the pairs' inner rows side by side, and of the tokens' own."""
    args, want = _experts(T, E, k, K, I, seed=k, missing=missing)
    assert _lib.lib().pxl_moe_mx4_few_takes(T, k, K, I) == 1
    first = ops.moe_ffn_mx4(**args)
    oracle.within(first, *want)
    with cu.launch_chain():
        again = [ops.moe_ffn_mx4(**args) for _ in range(3)]
    assert all(torch.equal(y, first) for y in again)


@pytest.mark.parametrize("T,E,k,K,I", [(1, 32, 4, 2880, 2880), (64, 128, 4, 2880, 320), (3001, 128, 8, 256, 192), (1100, 32, 4, 2880, 256)])
def test_experts_give_the_same_bits_on_every_run(T, E, k, K, I):
    """The order of an expert's rows may differ from run to run, their results may not."""
    g = torch.Generator(device=DEV).manual_seed(T)
    w1, w2 = (ops.Mx4Weight.pack(torch.randint(0, 256, (r, c // 2), generator=g, dtype=torch.uint8, device=DEV),
                                 torch.randint(112, 120, (r, c // 32), generator=g, dtype=torch.uint8, device=DEV), experts=E)
              for r, c in ((E * 2 * I, K), (E * K, I)))
    x = torch.randn(T, K, generator=g, device=DEV).bfloat16()
    ids = torch.rand(T, E, generator=g, device=DEV).topk(k).indices.int().contiguous()
    wts = torch.rand(T, k, generator=g, device=DEV)
    first = ops.moe_ffn_mx4(x, ids, wts, w1, w2, base=x)
    for _ in range(20):
        assert torch.equal(ops.moe_ffn_mx4(x, ids, wts, w1, w2, base=x), first)


@pytest.mark.parametrize("T", [1, 3, 70])
def test_a_result_in_the_place_of_its_residual(T):
    codes, scales = _matrix(192, 256, 1)
    w, x = ops.Mx4Weight.pack(codes.to(DEV), scales.to(DEV)), _normal(T, 256).to(DEV)
    buf = _normal(T, 400, seed=1).to(DEV)
    want = oracle.linear(x.cpu().double(), oracle.values(codes, scales), residual=buf[:, :192].cpu())
    kept = buf.clone()
    out = buf.view(-1)[:192].view(1, 192) if T == 1 else buf[:, :192]          # (of one row the strides may differ)
    oracle.within(ops.linear_mx4(x, w, residual=buf[:, :192], out=out), *want)
    assert torch.equal(buf[:, 192:], kept[:, 192:])


@pytest.mark.parametrize("T,N,K", [(5, 640, 4096), (60, 40000, 224), (130, 2800, 768), (300, 512, 1024), (1500, 1536, 512)])
def test_results_with_and_without_a_residual_of_zeros(T, N, K):
    """Results leave the kernel in another way beside a residual: the same bits."""
    (xc, xs), (wc, ws) = (tuple(t.to(DEV) for t in _matrix(r, K, r)) for r in (T, N))
    b = _normal(N, seed=1).to(DEV)
    want = ops.linear_mx4_rows(xc, xs, wc, ws, b)
    assert torch.equal(ops.linear_mx4_rows(xc, xs, wc, ws, b, residual=torch.zeros_like(want)), want)
    wide = torch.zeros(T, N + 3, dtype=torch.bfloat16, device=DEV)             # and to rows that start on no 16 bytes
    assert torch.equal(ops.linear_mx4_rows(xc, xs, wc, ws, b, out=wide[:, 3:]), want)
