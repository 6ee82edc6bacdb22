"""optimizer "muon" and the 8-bit layers in the training engine, on the CPU (single process and gloo ranks)."""
import pytest
import torch

from dllm.models import reference as R
from dllm.models.ffn import init_ffn_layer, layer_bwd_fp8, layer_fwd_fp8
from dllm.ops import fp8, muon
from dllm.parallel.engine import FFNTrainer
from dllm.parallel.mesh import Mesh
from dllm.utils.config import ModelConfig, TrainConfig
from dllm.utils.data import reference_mock_data
from dllm.utils.sizing import plan
from test_distributed_cpu import _run
from test_muon_cpu import exact

CPU = torch.device("cpu")


def _layers(D, F, L, gated=False, seed=3):
    gen = torch.Generator().manual_seed(seed)
    return [init_ffn_layer(D, F, gen, gated) for _ in range(L)]


def _muon_oracle(layers, batches, lr, wd, beta, nesterov, act):
    """The formula in 64 bits: summed gradients of each step's batches, momentum, orthogonalised update."""
    layers = [{k: v.double() for k, v in p.items()} for p in layers]
    mom = [{k: torch.zeros_like(v) for k, v in p.items()} for p in layers]
    for step in batches:
        total = None
        for x, dy in step:
            _, g = R.stack_grads(layers, x.double(), dy.double(), act)
            total = g if total is None else [{k: a[k] + b[k] for k in a} for a, b in zip(total, g)]
        for p, m, g in zip(layers, mom, total):
            for k in p:
                m[k] = beta * m[k] + g[k]
                u = g[k] + beta * m[k] if nesterov else m[k]
                p[k] = (1 - lr * wd) * p[k] - lr * muon.muon_scale(*p[k].shape) * exact(u)
    return layers


@pytest.mark.parametrize("act,gated,nesterov", [("relu", False, True), ("gelu", False, False), ("silu", True, True)])
def test_muon_engine_matches_formula(act, gated, nesterov):
    D, F, T, L, lr, wd = 16, 32, 24, 2, 0.02, 0.1
    layers = _layers(D, F, L, gated)
    batches = [[b] for b in reference_mock_data([5, 6], T, D)]
    cfg = TrainConfig(model=ModelConfig(D, F, L, act, gated), batch_size=1, seq_len=T, lr=lr, optimizer="muon",
                      weight_decay=wd, muon_beta=0.9, muon_nesterov=nesterov)
    eng = FFNTrainer(cfg, Mesh(), CPU)
    eng.load_full_params(layers)
    for (x, dy), in batches:
        eng.train_step(x, dy)
    want = _muon_oracle(layers, batches, lr, wd, 0.9, nesterov, act)
    for g, w in zip(eng.gather_full_params(), want):
        for k in w:
            # two steps; each update is exact to 3e-4 of its largest singular value (see test_muon_cpu.TOL), which bounds the
            # elements: at most 1.25 * 2 (tall scale sqrt(2)) * lr, and the second step's gradient sees the first's error
            assert (g[k].double() - w[k]).abs().max() <= 4 * 3e-4 * 1.25 * 1.5 * lr, k


def test_muon_ddp_equals_formula(free_port):
    """Two gloo ranks: the update of the summed gradient, identical on both."""
    cfg = TrainConfig(model=ModelConfig(8, 16, 2), batch_size=1, seq_len=16, num_steps=4, lr=0.02, optimizer="muon",
                      data="cpu_compat")
    layers = _layers(8, 16, 2)
    seeds = [11, 12, 13, 14]
    got = _run(cfg, 2, 2, free_port, params=layers, seeds=seeds)
    data = list(reference_mock_data(seeds, 16, 8))
    want = _muon_oracle(layers, [data[0:2], data[2:4]], 0.02, 0.0, 0.95, True, "relu")
    for g, w in zip(got, want):
        for k in w:
            assert (g[k].double() - w[k]).abs().max() <= 4 * 3e-4 * 1.25 * 1.5 * 0.02, k


def test_muon_checkpoint_resume(tmp_path, free_port):
    cfg = TrainConfig(model=ModelConfig(8, 16, 2), batch_size=1, seq_len=16, num_steps=4, lr=0.02, optimizer="muon",
                      data="cpu_compat")
    for fmt in ("consolidated", "sharded"):
        ck = str(tmp_path / fmt)
        full = _run(cfg, 2, 2, free_port)
        _run(cfg, 2, 2, free_port + 1, ckpt_dir=ck, stop_after=1, ckpt_format=fmt)
        resumed = _run(cfg, 2, 2, free_port + 2, resume=ck)
        for g, w in zip(resumed, full):
            for k in w:
                torch.testing.assert_close(g[k], w[k], rtol=1e-6, atol=1e-8)


@pytest.mark.parametrize("opt", ["sgd", "muon"])
@pytest.mark.parametrize("act", ["relu", "silu"])
@pytest.mark.parametrize("grad_dtype", ["fp32", "bf16"])
def test_fp8_engine_step_is_its_operators(opt, act, grad_dtype):
    """One step of a two-layer stack equals the layer functions and the optimizer called by hand."""
    D, F, T, lr = 24, 40, 20, 0.01
    layers = _layers(D, F, 2)
    (x, dy), = list(reference_mock_data([7], T, D))
    x, dy = x.bfloat16(), dy.bfloat16()
    cfg = TrainConfig(model=ModelConfig(D, F, 2, act), batch_size=1, seq_len=T, lr=lr, dtype="bf16", optimizer=opt, fp8=True,
                      grad_dtype=grad_dtype, master="fp32")
    eng = FFNTrainer(cfg, Mesh(), CPU)
    eng.load_full_params(layers)
    y = eng.train_step(x, dy)
    gd = cfg.torch_grad_dtype
    acts, saved, inp = [], [], x
    for p in layers:
        w1, w2 = p["w1"].bfloat16(), p["w2"].bfloat16()
        a, h, out = (torch.empty(T, n, dtype=torch.bfloat16) for n in (F, F, D))
        saved.append(layer_fwd_fp8(inp, w1, w2, act, a, None if act == "relu" else h, out))
        acts.append((a, None if act == "relu" else h))
        inp = out
    assert torch.equal(y, inp)
    g = dy
    for i in (1, 0):
        w1, w2 = layers[i]["w1"].bfloat16(), layers[i]["w2"].bfloat16()
        g1, g2 = torch.empty(F, D, dtype=gd), torch.empty(D, F, dtype=gd)
        g = layer_bwd_fp8(g, saved[i], w1, w2, act, *acts[i], g1, g2, torch.empty(T, F, dtype=torch.bfloat16),
                          torch.empty(T, D, dtype=torch.bfloat16) if i else None)
        for k, gw in (("w1", g1), ("w2", g2)):
            w = layers[i][k].clone()
            if opt == "sgd":
                w.add_(-lr * gw.float())
            else:
                muon.muon_step_(w, gw, torch.zeros_like(w), lr=lr)
            assert torch.equal(eng.gather_full_params()[i][k], w), (i, k)


def test_fp8_layer_against_unquantised():
    """The 8-bit layer's outputs and gradients against 64-bit arithmetic on the same inputs: every product has two operands
    rounded by at most 2^-4 (e4m3) or 2^-3 (e5m2) of themselves (plus what falls below 2^-9 / 2^-16 of the block's largest
    code, 2^-17 / 2^-31 of the block's maximum), so |error| <= bound * sum|a||b| per product; bf16 outputs add 2^-8."""
    gen = torch.Generator().manual_seed(1)
    T, D, F = 30, 20, 36
    x, dy = torch.randn(T, D, generator=gen).bfloat16(), torch.randn(T, D, generator=gen).bfloat16()
    w1, w2 = (0.2 * torch.randn(F, D, generator=gen)).bfloat16(), (0.2 * torch.randn(D, F, generator=gen)).bfloat16()
    a, y, da = (torch.empty(T, n, dtype=torch.bfloat16) for n in (F, D, F))
    saved = layer_fwd_fp8(x, w1, w2, "relu", a, None, y)
    g1, g2, dx = torch.empty(F, D), torch.empty(D, F), torch.empty(T, D, dtype=torch.bfloat16)
    layer_bwd_fp8(dy, saved, w1, w2, "relu", a, None, g1, g2, da, dx)

    def near(got, p, q, b, where=True):
        p, q = p.double(), q.double()
        mag = p.abs() @ q.abs().t()
        err = (got.double() - p @ q.t()).abs()
        assert (torch.where(torch.as_tensor(where), err, 0.0) <= b * mag + 2 ** -8 * mag + 1e-4 * mag.max()).all()

    e4, e5 = 2 ** -4, 2 ** -3
    h = (x.double() @ w1.double().t())
    bound = (2 * e4 + e4 ** 2 + 2 ** -8) * (x.double().abs() @ w1.double().abs().t()) + 1e-4 * h.abs().max()
    assert ((a.double() - h.clamp(min=0)).abs() <= bound).all()
    near(y, a, w2, 2 * e4 + e4 ** 2)
    live = a > 0                                       # the mask of the stored activation
    assert (da[~live] == 0).all()
    near(da, dy, w2.t(), e4 + e5 + e4 * e5, live)
    near(dx, da, w1.t(), e4 + e5 + e4 * e5)
    near(g2, dy.t(), a.t(), e4 + e5 + e4 * e5)
    near(g1, da.t(), x.t(), e4 + e5 + e4 * e5)


@pytest.mark.parametrize("method", [2, 3, 6])
def test_fp8_data_parallel_modes_agree(method, free_port):
    """DDP, FSDP and ZeRO-2 on two gloo ranks quantise the same tensors: FSDP and ZeRO equal DDP."""
    cfg = TrainConfig(model=ModelConfig(16, 32, 3), batch_size=1, seq_len=16, num_steps=2, lr=1e-2, dtype="bf16", fp8=True,
                      grad_dtype="fp32", data="cpu_compat")
    want = _run(cfg, 2, 2, free_port)
    got = _run(cfg, method, 2, free_port + 1)
    for g, w in zip(got, want):
        for k in w:
            torch.testing.assert_close(g[k], w[k], rtol=0, atol=0)


def test_refusals():
    def build(mesh=None, **kw):
        m = {"model": ModelConfig(16, 32, 1, gated=kw.pop("gated", False)), "batch_size": 1, "seq_len": 16}
        return FFNTrainer(TrainConfig(**m, **kw), mesh or Mesh(), CPU)

    with pytest.raises(ValueError, match="unknown optimizer"):
        build(optimizer="lion")
    for kw in ({"dp_mode": "zero", "force_comm": True}, {"dp_mode": "fsdp", "force_comm": True}):
        with pytest.raises(ValueError, match="whole weight matrices"):
            build(optimizer="muon", **kw)
    with pytest.raises(ValueError, match="fp8 needs dtype bf16"):
        build(fp8=True)
    with pytest.raises(ValueError, match="ungated"):
        build(fp8=True, dtype="bf16", gated=True)
    with pytest.raises(ValueError, match="recompute none"):
        build(fp8=True, dtype="bf16", recompute="full")
    with pytest.raises(ValueError, match="row-major"):
        build(fp8=True, dtype="bf16", w2_storage="transposed")
    with pytest.raises(ValueError, match="wgrad_layout"):
        build(fp8=True, dtype="bf16", wgrad_layout="nn")


def test_interleaved_weight_is_two_matrices():
    gen = torch.Generator().manual_seed(4)
    w, g, m = (torch.randn(64, 10, generator=gen) for _ in range(3))
    w2, m2 = w.clone(), m.clone()
    muon.muon_step_(w, g, m, lr=0.1, wd=0.1, interleave=16)
    pick = lambda t, i: torch.cat([t[32 * k + 16 * i:32 * k + 16 * i + 16] for k in range(2)])  # noqa: E731
    for i in range(2):
        wi, mi = pick(w2, i), pick(m2, i)
        muon.muon_step_(wi, pick(g, i), mi, lr=0.1, wd=0.1)
        torch.testing.assert_close(pick(w, i), wi, rtol=1e-5, atol=1e-6)
        assert torch.equal(pick(m, i), mi)
    with pytest.raises(ValueError, match="interleave"):
        muon.muon_step_(w[:60].clone(), g[:60].clone(), m[:60].clone(), lr=0.1, interleave=16)


def test_sizing_knows_both():
    base = plan(512, 2048, 4, 1024)
    mu = plan(512, 2048, 4, 1024, optimizer="muon")
    assert mu["bytes"]["muon_momentum"] == 4 * mu["params_per_rank"] and mu["bytes"]["grads"] > 0 == base["bytes"]["grads"]
    f8 = plan(512, 2048, 4, 1024, fp8=True)
    assert f8["bytes"]["fp8_saved"] > 0 and "nn_transposed_copies" not in f8["bytes"]


def test_cli_takes_both():
    from dllm.train_ffns import config_from_args, make_parser

    cfg = config_from_args(make_parser().parse_args(["--optimizer", "muon", "--muon_beta", "0.9", "--fp8", "--dtype", "bf16"]))
    assert cfg.optimizer == "muon" and cfg.muon_beta == 0.9 and cfg.fp8
    assert fp8.BLOCK == 128


@pytest.mark.parametrize("act,gated", [("relu", False), ("silu", True)])
@pytest.mark.parametrize("D,F", [(16, 32), (32, 16)])
def test_muon_on_transposed_w2_storage(act, gated, D, F):
    """W2 kept as W2ᵀ: the same update (scale by the logical shape), against the formula and in a checkpoint's logical form."""
    T, L, lr, wd = 24, 2, 0.02, 0.1
    layers = _layers(D, F, L, gated)
    batches = [[b] for b in reference_mock_data([5, 6], T, D)]
    cfg = TrainConfig(model=ModelConfig(D, F, L, act, gated), batch_size=1, seq_len=T, lr=lr, optimizer="muon", weight_decay=wd,
                      muon_beta=0.9, w2_storage="transposed")
    eng = FFNTrainer(cfg, Mesh(), CPU)
    assert eng.w2t
    eng.load_full_params(layers)
    for (x, dy), in batches:
        eng.train_step(x, dy)
    want = _muon_oracle(layers, batches, lr, wd, 0.9, True, act)
    for g, w in zip(eng.gather_full_params(), want):
        for k in w:
            # two steps, each off by 3e-4 of its largest singular value (at most 1.25), times the scale sqrt(2) and the learning rate
            assert g[k].shape == w[k].shape and (g[k].double() - w[k]).abs().max() <= 4 * 3e-4 * 1.25 * 1.5 * lr, k
    mom = eng.gather_full_params(eng.muon_m)
    assert all(m["w2"].shape == (D, F) for m in mom)
