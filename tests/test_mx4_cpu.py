"""Microscaled 4-bit operators on the CPU: quantisation, the weights' layout, products, and what is refused."""

import pytest
import torch

from parallax_b200 import ops
from parallax_b200.loader.quant import dequant_mxfp4
from tests.helpers import mx4_oracle as oracle


def _matrix(rows, K, seed, lo=120, hi=128):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 256, (rows, K // 2), generator=g, dtype=torch.uint8),
            torch.randint(lo, hi, (rows, K // 32), generator=g, dtype=torch.uint8))


def _borders():
    """Every border between two numbers and its neighbours in fp32, and their negatives."""
    b = (oracle.MAGS[1:] + oracle.MAGS[:-1]) / 2
    b = torch.cat([b, oracle.MAGS]).float()
    v = torch.cat([b, torch.nextafter(b, torch.tensor(float("inf"))), torch.nextafter(b, torch.tensor(-float("inf")))])
    v = torch.cat([v, -v])
    return torch.nn.functional.pad(v[v.abs() <= 6], (0, 0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 96), (17, 416)])
def test_quantisation(rows, K, dtype):
    x = (torch.randn(rows, K, generator=torch.Generator().manual_seed(rows)) * 3.0).to(dtype)
    want, e, _fine = oracle.quantise(x)
    codes, scales = ops.quant_mx4_rows(x)
    assert torch.equal(scales.double() - 127, e)
    assert torch.equal(oracle.values(codes, scales), want)
    assert torch.equal(ops.expand_mx4_rows(codes, scales).double(), want)


def test_quantisation_on_borders_and_extremes():
    v = _borders()
    rows = []
    for power in (-126, -30, 0, 17, 120):
        for i in range(0, v.numel(), 31):
            part = v[i:i + 31]
            rows.append(torch.cat([part, torch.tensor([6.0]), torch.zeros(31 - part.numel())]) * 2.0 ** power)
    for most in (3.0, 3.0000002, 6.0, 6.0000005, 1.5, 5.9999995):
        rows.append(torch.full((32,), most))
    rows += [torch.zeros(32), torch.full((32,), 2.0 ** -149), torch.full((32,), 2.0 ** -127), torch.full((32,), 3e38), torch.full((32,), -0.0)]
    x = torch.stack(rows)
    want, e, _fine = oracle.quantise(x)
    codes, scales = ops.quant_mx4_rows(x)
    assert torch.equal(scales.double() - 127, e) and torch.equal(oracle.values(codes, scales), want)


def test_groups_with_nan_or_infinity():
    x = torch.randn(3, 64)
    x[0, 5], x[1, 40], x[2, 63] = float("nan"), float("inf"), -float("inf")
    codes, scales = ops.quant_mx4_rows(x)
    assert (scales == 255).tolist() == [[True, False], [False, True], [False, True]]
    v = ops.expand_mx4_rows(codes, scales)
    assert torch.equal(torch.isnan(v), (scales == 255).repeat_interleave(32, 1))
    assert int(codes[0, :16].max()) == 0


def test_values_are_those_of_the_checkpoint_format():
    codes, scales = _matrix(5, 128, 0, 0, 254)
    want = dequant_mxfp4(codes.view(5, 4, 16), scales, torch.float32)
    assert torch.equal(ops.expand_mx4_rows(codes, scales), want.bfloat16())
    assert torch.equal(oracle.values(codes, scales).float(), want)


@pytest.mark.parametrize("experts,N,K", [(1, 1, 32), (1, 130, 160), (3, 128, 128), (2, 300, 96), (1, 257, 1056)])
def test_layout_gives_back_what_went_in(experts, N, K):
    codes, scales = _matrix(experts * N, K, N, 0, 129)
    w = ops.Mx4Weight.pack(codes, scales, experts=experts)
    c, s = w.unpack()
    assert torch.equal(c, codes) and torch.equal(s, scales)
    assert float(w.row_scale.min()) == float(w.row_scale.max()) == 1.0
    if experts > 1:
        c, s = w.expert_slice(1, 2).unpack()
        assert torch.equal(c, codes[N:2 * N]) and torch.equal(s, scales[N:2 * N])


def test_layout_in_parts_equals_the_whole(monkeypatch):
    from parallax_b200.ops import mx4

    codes, scales = _matrix(700, 288, 5)
    whole = ops.Mx4Weight.pack(codes, scales)
    monkeypatch.setattr(mx4, "_CHUNK", 1)
    part = ops.Mx4Weight.pack(codes, scales)
    assert torch.equal(whole.data, part.data) and torch.equal(whole.row_scale, part.row_scale)


def test_layout_of_large_and_nan_scales():
    codes, scales = _matrix(6, 96, 1)
    scales[0, 1], scales[1, 0], scales[2, 2], scales[3, 1], scales[3, 2] = 254, 129, 255, 255, 200
    w = ops.Mx4Weight.pack(codes, scales)
    f = w.row_scale[0, :6]
    assert float(f[0]) == 2.0 ** 126 and float(f[1]) == 2.0 and torch.isnan(f[2:4]).all() and float(f[4]) == 1.0
    c, s = w.unpack()
    assert torch.equal(s[1:3], scales[1:3]) and torch.equal(c[1:3], codes[1:3]) and torch.equal(s[4:], scales[4:])
    assert torch.equal(s[3] == 255, scales[3] == 255)
    assert int(s[0, 1]) == 254 and torch.equal(c[0, 16:32], codes[0, 16:32]) and int(c[0, :16].max()) == 0     # 2^128 below 2^127


@pytest.mark.parametrize("T,N,K", [(0, 64, 32), (1, 3, 32), (5, 200, 160)])
def test_products(T, N, K):
    g = torch.Generator().manual_seed(N)
    x = torch.randn(T, K, generator=g).bfloat16()
    codes, scales = _matrix(N, K, 3)
    bias, res = torch.randn(N, generator=g).bfloat16(), torch.randn(T, N, generator=g).bfloat16()
    w, wide = ops.Mx4Weight.pack(codes, scales), oracle.values(codes, scales)
    for b, r in ((None, None), (bias, None), (bias, res)):
        oracle.within(ops.linear_mx4(x, w, bias=b, residual=r), *oracle.linear(x.double(), wide, b, r))
    out = torch.empty(T, N, dtype=torch.bfloat16)
    assert ops.linear_mx4(x, w, out=out) is out
    xc, xs = ops.quant_mx4_rows(x)
    oracle.within(ops.linear_mx4_rows(xc, xs, codes, scales, bias=bias, residual=res),
                  *oracle.linear(oracle.values(xc, xs), wide, bias, res))


@pytest.mark.parametrize("clip", [False, True])
def test_experts(clip):
    E, I, K, T, k = 4, 64, 96, 9, 2
    g = torch.Generator().manual_seed(7)
    x, base = torch.randn(T, K, generator=g).bfloat16(), torch.randn(T, K, generator=g).bfloat16()
    (c1, s1), (c2, s2) = _matrix(E * 2 * I, K, 1), _matrix(E * K, I, 2)
    b1, b2 = torch.randn(E, 2 * I, generator=g).bfloat16(), torch.randn(E, K, generator=g).bfloat16()
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).int()
    ids[3] = torch.tensor([1, 1])                   # the same expert twice
    ids[4] = torch.tensor([-1, E])                  # none of them
    wts = torch.rand(T, k, generator=g)
    got = ops.moe_ffn_mx4(x, ids, wts, ops.Mx4Weight.pack(c1, s1, E), ops.Mx4Weight.pack(c2, s2, E), base=base, act_mode=int(clip),
                          limit=2.0, b1=b1.flatten(), b2=b2.flatten())
    want = oracle.experts(x, ids, wts, oracle.values(c1, s1).view(E, 2 * I, K), oracle.values(c2, s2).view(E, K, I), base, clip, 2.0, b1, b2)
    oracle.within(got, *want)
    assert torch.equal(got[4], base[4])


def test_gate_matches_the_dense_experts():
    """The same model as moe_ffn over the expanded matrices."""
    E, I, K, T = 3, 64, 64, 5
    (c1, s1), (c2, s2) = _matrix(E * 2 * I, K, 1), _matrix(E * K, I, 2)
    x, ids, wts = torch.randn(T, K), torch.randint(0, E, (T, 2)).int(), torch.rand(T, 2)
    w1, w2 = oracle.values(c1, s1).float(), oracle.values(c2, s2).float()
    a = ops.moe_ffn_mx4(x, ids, wts, ops.Mx4Weight.pack(c1, s1, E), ops.Mx4Weight.pack(c2, s2, E))
    b = ops.moe_ffn(x, ids, wts, w1, w2, E)
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-4 * float(b.abs().max()))


def _expert_call(**kw):
    E, I, K, T = 2, 64, 64, 3
    a = dict(x=torch.zeros(T, K, dtype=torch.bfloat16), ids=torch.zeros(T, 2, dtype=torch.int32), weights=torch.ones(T, 2),
             w1=ops.Mx4Weight.pack(*_matrix(E * 2 * I, K, 1), E), w2=ops.Mx4Weight.pack(*_matrix(E * K, I, 2), E))
    a.update(kw)
    return ops.moe_ffn_mx4(**a)


@pytest.mark.parametrize("kw", [
    dict(ids=torch.zeros(3, 2, dtype=torch.int64)), dict(ids=torch.zeros(2, 2, dtype=torch.int32)), dict(weights=torch.ones(3, 1)),
    dict(weights=torch.ones(3, 2).bfloat16()), dict(base=torch.zeros(2, 64).bfloat16()), dict(base=torch.zeros(3, 64)), dict(act_mode=2),
    dict(act_mode=1, limit=0.0), dict(b1=torch.zeros(5).bfloat16()), dict(b2=torch.zeros(2 * 64)),
    dict(w1=ops.Mx4Weight.pack(*_matrix(2 * 64, 64, 1), 2)), dict(w2=ops.Mx4Weight.pack(*_matrix(64, 64, 1), 1)),
    dict(x=torch.zeros(3, 96).bfloat16())])
def test_experts_refuse(kw):
    assert _expert_call().shape == (3, 64)
    with pytest.raises(ops.KernelError):
        _expert_call(**kw)


def test_results_that_share_memory():
    """Refused, but for a residual's own place and other columns of the rows' buffer."""
    codes, scales = _matrix(128, 128, 0)
    w = ops.Mx4Weight.pack(codes, scales)
    buf = torch.randn(6, 384, generator=torch.Generator().manual_seed(0)).bfloat16()
    x, y = buf[:, :128], buf[:, 128:256]
    want = ops.linear_mx4(x, w)
    assert torch.equal(ops.linear_mx4(x, w, out=y), want) and torch.equal(y, want)
    assert torch.equal(ops.linear_mx4(x[1:], w, out=buf[:5, 256:]), want[1:])
    r = torch.randn(6, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    want = ops.linear_mx4(x, w, residual=r)
    assert torch.equal(ops.linear_mx4(x, w, residual=r, out=r), want) and torch.equal(r, want)
    flat = torch.zeros(2000, dtype=torch.bfloat16)
    for call in (lambda: ops.linear_mx4(x, w, out=x), lambda: ops.linear_mx4(x, w, out=buf[:, 64:192]),
                 lambda: ops.linear_mx4(buf[:, 256:], w, out=buf[:, 192:320]), lambda: ops.linear_mx4(x[:3], w, out=x[2:5]),
                 lambda: ops.linear_mx4(x, w, residual=flat[:768].view(6, 128), out=flat[128:896].view(6, 128)),
                 lambda: ops.linear_mx4(x, w, residual=flat[:768].view(6, 128), out=flat[:1536].view(6, 256)[:, :128])):
        with pytest.raises(ops.KernelError):
            call()


def test_refusals():
    codes, scales = _matrix(128, 64, 0)
    w, x = ops.Mx4Weight.pack(codes, scales), torch.zeros(2, 64, dtype=torch.bfloat16)
    two = ops.Mx4Weight.pack(codes, scales, experts=2)
    bad = [
        lambda: ops.quant_mx4_rows(torch.zeros(2, 48)), lambda: ops.quant_mx4_rows(torch.zeros(2, 0)),
        lambda: ops.quant_mx4_rows(torch.zeros(64)), lambda: ops.quant_mx4_rows(torch.zeros(2, 64, dtype=torch.float16)),
        lambda: ops.expand_mx4_rows(codes, scales[:5]), lambda: ops.expand_mx4_rows(codes.int(), scales),
        lambda: ops.expand_mx4_rows(codes, scales[:, :1]), lambda: ops.Mx4Weight.pack(codes, scales, experts=3),
        lambda: ops.Mx4Weight.pack(codes[:0], scales[:0]), lambda: ops.Mx4Weight.pack(codes, scales, experts=0),
        lambda: ops.linear_mx4(torch.zeros(2, 96, dtype=torch.bfloat16), w), lambda: ops.linear_mx4(x, two),
        lambda: ops.linear_mx4(x, codes), lambda: ops.linear_mx4(x, w, epi=ops.EPI_F32),
        lambda: ops.linear_mx4(x, w, epi=ops.EPI_CLIP_GLU), lambda: ops.linear_mx4(x, w, bias=torch.zeros(64).bfloat16()),
        lambda: ops.linear_mx4(x, w, bias=torch.zeros(128)), lambda: ops.linear_mx4(x, w, residual=torch.zeros(2, 64).bfloat16()),
        lambda: ops.linear_mx4(x, w, epi=ops.EPI_SILU_MUL, residual=torch.zeros(2, 64).bfloat16()),
        lambda: ops.linear_mx4(x, w, epi=ops.EPI_RESIDUAL), lambda: ops.linear_mx4(x, w, out=torch.zeros(2, 64).bfloat16()),
        lambda: ops.linear_mx4(x, w, out=torch.zeros(128, 2).bfloat16().t()),
        lambda: ops.linear_mx4(x, ops.Mx4Weight.pack(codes[:120], scales[:120]), epi=ops.EPI_SILU_MUL),
        lambda: ops.linear_mx4_rows(codes, scales, codes[:, :16], scales[:, :1]),
        lambda: ops.linear_mx4_rows(codes, scales, codes, scales, bias=torch.zeros(64).bfloat16()),
        lambda: ops.linear_mx4_rows(codes.float(), scales, codes, scales),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ops.KernelError):
            call()
            pytest.fail(f"call {i} was not refused")


# ------------------------------------------------------------------------------------------------ engine
def _gpt_oss(hidden=128, inner=64):
    from parallax_b200.models.config import config_from_hf

    return config_from_hf(dict(
        architectures=["GptOssForCausalLM"], model_type="gpt_oss", hidden_size=hidden, num_hidden_layers=2, num_attention_heads=4,
        num_key_value_heads=2, head_dim=32, intermediate_size=inner, moe_intermediate_size=inner, num_local_experts=4, num_experts_per_tok=2, sliding_window=16,
        layer_types=["sliding_attention", "full_attention"], vocab_size=256, max_position_embeddings=512, rope_theta=10000.0,
        attention_bias=True, tie_word_embeddings=False))


def _checkpoint(cfg, seed=0):
    """Random weights of a small GPT-OSS under their published names, experts as MXFP4 blocks."""
    g = torch.Generator().manual_seed(seed)
    H, D, I, E = cfg.hidden_size, cfg.head_dim, cfg.moe_intermediate_size, cfg.num_experts
    rnd = lambda *sh: torch.randn(*sh, generator=g) * 0.1  # noqa: E731
    sd = {"model.embed_tokens.weight": rnd(cfg.vocab_size, H), "model.norm.weight": torch.ones(H), "lm_head.weight": rnd(cfg.vocab_size, H)}
    for i in range(cfg.num_hidden_layers):
        p, m = f"model.layers.{i}.", f"model.layers.{i}.mlp."
        for n in ("input_layernorm", "post_attention_layernorm"):
            sd[p + n + ".weight"] = torch.ones(H)
        for n, rows in (("q", 4 * D), ("k", 2 * D), ("v", 2 * D)):
            sd[p + f"self_attn.{n}_proj.weight"], sd[p + f"self_attn.{n}_proj.bias"] = rnd(rows, H), rnd(rows)
        sd[p + "self_attn.o_proj.weight"], sd[p + "self_attn.o_proj.bias"], sd[p + "self_attn.sinks"] = rnd(H, 4 * D), rnd(H), rnd(4)
        sd[m + "router.weight"], sd[m + "router.bias"] = rnd(E, H), rnd(E)
        for n, rows, cols in (("gate_up_proj", 2 * I, H), ("down_proj", H, I)):
            c, s = ops.quant_mx4_rows(rnd(E * rows, cols) * 3)
            sd[m + f"experts.{n}_blocks"], sd[m + f"experts.{n}_scales"] = c.view(E, rows, cols // 32, 16), s.view(E, rows, cols // 32)
            sd[m + f"experts.{n}_bias"] = rnd(E, rows)
    return sd


def _logits(cfg, weights, **kw):
    from parallax_b200.engine.engine import Engine
    from parallax_b200.engine.request import Request, SamplingParams

    eng = Engine(cfg, device="cpu", num_blocks=64, page_size=16, max_batch_size=4, weights=weights, **kw)
    eng.keep_logits = True
    req = Request(input_ids=list(range(3, 40)), sampling_params=SamplingParams(max_new_tokens=3, temperature=0.0, ignore_eos=True))
    eng.add_request(req)
    out = []
    while eng.has_work():
        eng.step()
        if eng.last_logits is not None and eng.last_logits.shape[0] > 0:
            out.append(eng.last_logits[0].clone())
        eng.last_logits = None
    return eng, torch.stack(out), req.output_ids


def test_engine_keeps_packed_experts():
    """The same model with its experts expanded and kept in 4 bits."""
    cfg = _gpt_oss()
    sd = _checkpoint(cfg)
    _eng, a, ta = _logits(cfg, sd)
    eng, b, tb = _logits(cfg, sd, expert_format="mxfp4")
    assert ta == tb and torch.allclose(a, b, rtol=1e-4, atol=1e-5)
    moe = eng.stages[0].model.layers[0].moe
    assert moe.w1 is None and moe.w2 is None and set(moe.mx4) == {"w1", "w2"}
    before = moe.mx4["w1"].data.data_ptr()
    other = _checkpoint(cfg, seed=1)
    eng.stages[0].model.reload_layers(other)                       # online refit moves new blocks into the same storage
    assert eng.stages[0].model.layers[0].moe.mx4["w1"].data.data_ptr() == before
    _e, c, tc = _logits(cfg, other)
    got = [lw.moe.mx4["w2"].unpack()[0] for lw in eng.stages[0].model.layers]
    for i, w in enumerate(got):
        assert torch.equal(w.view(-1), other[f"model.layers.{i}.mlp.experts.down_proj_blocks"].reshape(-1))


@pytest.mark.parametrize("clipped", [False, True])
def test_engine_quantises_experts_when_it_loads(clipped):
    """Random weights: the engine with 4-bit experts is the one whose experts hold the quantised values."""
    from parallax_b200.engine.engine import Engine
    from parallax_b200.models.config import config_from_hf

    cfg = _gpt_oss() if clipped else config_from_hf(dict(
        architectures=["Qwen3MoeForCausalLM"], model_type="qwen3_moe", hidden_size=128, num_hidden_layers=2, num_attention_heads=4,
        num_key_value_heads=2, head_dim=32, intermediate_size=128, moe_intermediate_size=64, num_experts=4, num_experts_per_tok=2,
        vocab_size=256, norm_topk_prob=True, rope_theta=1e4))
    plain = Engine(cfg, device="cpu", num_blocks=32, page_size=16, max_batch_size=2)
    packed = Engine(cfg, device="cpu", num_blocks=32, page_size=16, max_batch_size=2, expert_format="mxfp4")
    x = torch.randn(5, cfg.hidden_size)
    for lp, lq in zip(plain.stages[0].model.layers, packed.stages[0].model.layers):
        for name in ("w1", "w2"):
            w = getattr(lp.moe, name)
            w.copy_(ops.expand_mx4_rows(*ops.quant_mx4_rows(w)))
        assert torch.allclose(lp.moe.forward(x, x), lq.moe.forward(x, x), rtol=1e-4, atol=1e-5)


def test_engine_refuses():
    from parallax_b200.engine.engine import Engine
    from parallax_b200.models.config import named_config

    for cfg, fmt in ((named_config("tiny"), "mxfp4"), (_gpt_oss(), "int4"), (_gpt_oss(inner=96), "mxfp4")):
        with pytest.raises(ValueError):
            Engine(cfg, device="cpu", num_blocks=16, expert_format=fmt)
    moe = Engine(_gpt_oss(), device="cpu", num_blocks=16, expert_format="mxfp4").stages[0].model.layers[0].moe
    with pytest.raises(ValueError):
        moe.shard_experts(0, 2)


def test_launcher_refuses_several_processes():
    from parallax_b200.args import parse_args
    from parallax_b200.launch import run_scheduler_mode, run_standalone

    args = parse_args(["--model-path", "tiny-moe", "--random-init", "--expert-format", "mxfp4", "--pp-size", "2"])
    for run in (run_standalone, run_scheduler_mode):
        with pytest.raises(ValueError):
            run(args)
