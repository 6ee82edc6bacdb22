"""The quantiser, the 8-bit products and the Muon step together, as a training step uses them, on the GPU."""
import pytest
import torch

from dllm.models.ffn import init_ffn_layer, layer_bwd_fp8, layer_fwd_fp8
from dllm.ops import muon
from dllm.ops.elementwise import sgd_step_
from dllm.parallel.engine import FFNTrainer
from dllm.parallel.mesh import Mesh
from dllm.utils.config import ModelConfig, TrainConfig
from dllm.utils.graphs import GraphedStep

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _layers(D, F, L, gated=False, seed=3):
    gen = torch.Generator().manual_seed(seed)
    return [init_ffn_layer(D, F, gen, gated) for _ in range(L)]


def _data(T, D, seed=7):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(T, D, generator=g).bfloat16().to(DEV) for _ in range(2))


def _by_hand(layers, x, dy, act, lr, opt, gd):
    """Forward, backward and update of the stack from the operators; returns y and the new fp32 weights."""
    T, D, F = x.shape[0], x.shape[1], layers[0]["w1"].shape[0]
    layers = [{k: v.to(DEV) for k, v in p.items()} for p in layers]
    work = [{k: v.bfloat16() for k, v in p.items()} for p in layers]
    new = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    acts, saved, inp = [], [], x
    for w in work:
        a, h, out = new(T, F), None if act == "relu" else new(T, F), new(T, D)
        saved.append(layer_fwd_fp8(inp, w["w1"], w["w2"], act, a, h, out))
        acts.append((a, h))
        inp = out
    g = dy
    for i in reversed(range(len(work))):
        g1, g2 = (torch.empty(s, dtype=gd, device=DEV) for s in ((F, D), (D, F)))
        g = layer_bwd_fp8(g, saved[i], work[i]["w1"], work[i]["w2"], act, *acts[i], g1, g2, new(T, F), new(T, D) if i else None)
        for k, gw in (("w1", g1), ("w2", g2)):
            w = layers[i][k]
            if opt == "sgd":
                sgd_step_(w, gw, lr)
            else:
                muon.muon_step_(w, gw, torch.zeros_like(w), lr=lr)
    return inp, layers


@pytest.mark.parametrize("T,D,F", [(64, 128, 512), (300, 136, 328), (1, 64, 256), (1024, 512, 2048)])
@pytest.mark.parametrize("act", ["relu", "gelu"])
@pytest.mark.parametrize("opt", ["sgd", "muon"])
def test_engine_step_is_its_operators(T, D, F, act, opt):
    layers, (x, dy) = _layers(D, F, 2), _data(T, D)
    cfg = TrainConfig(model=ModelConfig(D, F, 2, act), batch_size=1, seq_len=T, lr=0.01, dtype="bf16", optimizer=opt, fp8=True,
                      grad_dtype="fp32", master="fp32")
    eng = FFNTrainer(cfg, Mesh(), torch.device(DEV))
    eng.load_full_params(layers)
    y = eng.train_step(x, dy).clone()
    want_y, want = _by_hand(layers, x, dy, act, 0.01, opt, torch.float32)
    assert torch.equal(y, want_y)
    for g, w in zip(eng.gather_full_params(), want):
        for k in w:
            assert torch.equal(g[k].to(DEV), w[k]), k


@pytest.mark.parametrize("fp8,gated", [(True, False), (False, False), (False, True)])
@pytest.mark.parametrize("master", ["fp32", "split"])
def test_muon_engine_masters_agree(fp8, gated, master):
    """Split and fp32 masters, batched W13: one weight's step equals the operator called on that weight alone."""
    D, F, T = 128, 256, 96
    layers, (x, dy) = _layers(D, F, 1, gated), _data(T, D)
    cfg = TrainConfig(model=ModelConfig(D, F, 1, "silu", gated), batch_size=1, seq_len=T, lr=0.01, dtype="bf16",
                      optimizer="muon", fp8=fp8, grad_dtype="fp32", master=master, weight_decay=0.1)
    eng = FFNTrainer(cfg, Mesh(), torch.device(DEV))
    eng.load_full_params(layers)
    eng.train_step(x, dy)
    m = eng.gather_full_params(eng.muon_m)[0]      # after one step from zero: the gradient
    got = eng.gather_full_params()[0]
    for k, w0 in layers[0].items():
        w, mom = w0.to(DEV), torch.zeros_like(w0, device=DEV)
        muon.muon_step_(w, m[k].to(DEV), mom, lr=0.01, wd=0.1)
        assert torch.equal(got[k].to(DEV), w), k


def test_muon_interleaved_equals_separate():
    g = torch.Generator().manual_seed(5)
    for R, C, il in ((512, 96, 16), (96, 200, 1), (64, 9, 1), (900, 301, 3), (640, 256, 64)):
        w, gr, m = (torch.randn(R, C, generator=g).to(DEV) for _ in range(3))
        pick = lambda t, i: t.view(-1, 2, il, C)[:, i].reshape(-1, C).contiguous()  # noqa: E731
        parts = [[pick(t, i) for t in (w, gr, m)] for i in range(2)]
        cp = torch.empty(R, C, dtype=torch.bfloat16, device=DEV)
        muon.muon_step_(w, gr, m, lr=0.1, wd=0.1, interleave=il, copy=cp)
        assert torch.equal(cp, w.bfloat16())
        for i, (wi, gi, mi) in enumerate(parts):
            muon.muon_step_(wi, gi, mi, lr=0.1, wd=0.1)
            assert torch.equal(pick(w, i), wi) and torch.equal(pick(m, i), mi)


def test_step_captured_and_replayed():
    """Quantise, products, backward and Muon of one layer in a graph: every replay equals the eager step, with eager work of
    the same operators and synchronisations between the replays."""
    T, D, F = 200, 136, 264
    layer = {k: v.to(DEV) for k, v in _layers(D, F, 1)[0].items()}
    x, dy = _data(T, D)

    def state():
        return {"w": {k: v.clone() for k, v in layer.items()}, "m": {k: torch.zeros_like(v) for k, v in layer.items()},
                "c": {k: v.bfloat16() for k, v in layer.items()}, "y": torch.empty(T, D, dtype=torch.bfloat16, device=DEV)}

    def step(s):
        a, h, da = (torch.empty(T, F, dtype=torch.bfloat16, device=DEV) for _ in range(3))
        saved = layer_fwd_fp8(x, s["c"]["w1"], s["c"]["w2"], "gelu", a, h, s["y"])
        g1, g2 = torch.empty(F, D, device=DEV), torch.empty(D, F, device=DEV)
        layer_bwd_fp8(dy, saved, s["c"]["w1"], s["c"]["w2"], "gelu", a, h, g1, g2, da, torch.empty_like(x))
        for k, g in (("w1", g1), ("w2", g2)):
            muon.muon_step_(s["w"][k], g, s["m"][k], lr=0.02, copy=s["c"][k])

    eager, graphed = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(graphed)
    for _ in range(4):
        graph.replay()
        step(eager)
        torch.cuda.synchronize()
        for part in ("w", "m", "c"):
            for k in layer:
                assert torch.equal(eager[part][k], graphed[part][k]), (part, k)
        assert torch.equal(eager["y"], graphed["y"])
        x.copy_(torch.randn(T, D, device=DEV))


@pytest.mark.parametrize("kw", [{"optimizer": "muon"}, {"fp8": True}, {"optimizer": "muon", "fp8": True}])
def test_side_stream_optimizer_agrees(kw):
    """The update on the side stream (side_optimizer -1) equals the update in order, over steps that reuse the buffers."""
    layers = _layers(128, 256, 3)
    res = []
    for side in (0, -1):
        cfg = TrainConfig(model=ModelConfig(128, 256, 3), batch_size=1, seq_len=64, lr=0.01, dtype="bf16", side_optimizer=side,
                          grad_dtype="fp32", **kw)
        eng = FFNTrainer(cfg, Mesh(), torch.device(DEV))
        eng.load_full_params(layers)
        for seed in range(3):
            eng.train_step(*_data(64, 128, seed))
        torch.cuda.synchronize()
        res.append(eng.gather_full_params())
    for a, b in zip(*res):
        assert all(torch.equal(a[k], b[k]) for k in a)


def test_graphed_step_refuses():
    for kw in ({"optimizer": "muon"}, {"fp8": True}):
        cfg = TrainConfig(model=ModelConfig(128, 256, 1), batch_size=1, seq_len=64, lr=0.01, dtype="bf16", **kw)
        eng = FFNTrainer(cfg, Mesh(), torch.device(DEV))
        with pytest.raises(ValueError):
            GraphedStep(eng, 64, 128)


@pytest.mark.parametrize("D,F", [(2048, 8192), (8192, 2048)])
@pytest.mark.parametrize("master", ["split", "fp32"])
def test_muon_on_transposed_w2_storage(D, F, master):
    """What a bf16 run of large weights does by itself: W2 stored as W2ᵀ.  One step against the iteration in 64 bits on the
    engine's own gradient (its momentum after one step from zero)."""
    from test_muon_step_gpu import iteration, norm, step_tolerance

    T, lr = 512, 0.05
    layers, (x, dy) = _layers(D, F, 1), _data(T, D)
    cfg = TrainConfig(model=ModelConfig(D, F, 1), batch_size=1, seq_len=T, lr=lr, dtype="bf16", optimizer="muon",
                      grad_dtype="fp32", master=master, weight_decay=0.1, w2_storage="transposed")
    eng = FFNTrainer(cfg, Mesh(), torch.device(DEV))
    assert eng.w2t
    eng.load_full_params(layers)
    eng.train_step(x, dy)
    grads, got = eng.gather_full_params(eng.muon_m)[0], eng.gather_full_params()[0]
    for k, w0 in layers[0].items():
        u = grads[k].to(DEV).double() * (1 + 0.95)           # nesterov: g + beta * momentum, momentum = g
        o = iteration(u)
        rate = lr * muon.muon_scale(*w0.shape)
        want = w0.to(DEV).double() * (1 - lr * 0.1) - rate * o
        assert got[k].shape == w0.shape
        assert norm(got[k].to(DEV).double() - want) <= step_tolerance(u, o) * rate * norm(o) + 3 * 2.0 ** -24 * norm(want), k
