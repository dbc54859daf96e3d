"""The example decoder layer against a plain one in 64 bits on the dequantised weights and the values that its cache stands for."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("decoder_layer", os.path.join(ROOT, "examples", "decoder_layer.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _plain(torch, nn, ex, layer, caches, x, positions, news):
    """The layer in float64 on the CPU; keys and values as they are in the cache."""
    w = {n: nn.dequantize(t, layer.quant.ggml_type).double().cpu() for n, t in layer.weights.items()}
    x = x.double().cpu()

    def norm(v, n):
        return v / (v.square().mean(-1, keepdim=True) + n.epsilon).sqrt() * n.gain.double().cpu()

    q = norm((norm(x, layer.norms[0]) @ w["q"].t()).view(len(x), layer.heads, layer.dim), layer.norms[2])
    c, s = (t[positions.long()].double().cpu()[:, None] for t in (layer.cos, layer.sin))
    a, b = q.chunk(2, -1)
    q = torch.cat([a * c - b * s, b * c + a * s], -1)
    lengths, out, at = caches.lengths.tolist(), [], 0
    for i, n in enumerate(news):
        length, group = lengths[i], layer.heads // layer.kv_heads
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        k, v = nn.kv_cache_read(caches.data, caches.table[i:i + 1], ints([length]), starts=ints([0, length]), max_new=length, rows=length)
        k, v = (t.double().cpu().repeat_interleave(group, 1).transpose(0, 1) for t in (k, v))
        scores = q[at:at + n].transpose(0, 1) @ k.transpose(1, 2) / layer.dim ** 0.5
        hidden = torch.arange(length)[None] > torch.arange(length - n, length)[:, None]
        out.append((scores.masked_fill(hidden, -np.inf).softmax(-1) @ v).transpose(0, 1).reshape(n, -1))
        at += n
    h = x + torch.cat(out) @ w["o"].t()
    f = norm(h, layer.norms[1])
    gate = f @ w["gate"].t()
    return h + (gate * torch.sigmoid(gate) * (f @ w["up"].t())) @ w["down"].t()


def test_layer_over_prompts_decoding_and_eviction(gpu):
    """Each of the layer's projections is within 1e-3 of its row's largest value by the dense path's own contract; the rest adds 1e-5: four of them in
    a chain stay within 1e-2 of the output's 2-norm."""
    torch = gpu
    from gomlx_amd import nn
    ex = _example()
    layer = ex.Layer(512, 8, 2, 768, seed=3, positions=300)
    caches = ex.Caches(layer, 3, 160, 32)
    news = [100, 37, 1]
    starts = torch.tensor([0, 100, 137, 138], dtype=torch.int32, device="cuda")
    x = torch.randn(138, 512, device="cuda")
    positions = torch.cat([torch.arange(n) for n in news]).int().cuda()
    caches.lengths += torch.tensor(news, dtype=torch.int32, device="cuda")

    def check(x, positions, news, **how):
        y = ex.step(layer, caches, x, positions, **how)
        want = _plain(torch, nn, ex, layer, caches, x, positions, news)
        assert (y.double().cpu() - want).norm() <= 1e-2 * want.norm()
        return y

    y = check(x, positions, news, starts=starts, max_new=100)
    # every row of every query head has given away weights that add up to one
    heads = caches.accounts.sum().item()
    assert abs(heads - 138 * 8) < 1e-3 * 138 * 8
    h, position = y[[99, 136, 137]], torch.tensor(news, dtype=torch.int32, device="cuda")
    for i in range(4):
        caches.lengths += 1
        h = check(h / h.square().mean(-1, keepdim=True).sqrt(), position, [1, 1, 1])
        position += 1
        if i == 1:
            ex.shrink(caches, 40, 8)
            assert caches.lengths.tolist() == [40, 39, 3]


def test_example_runs(gpu, monkeypatch, capsys):
    ex = _example()
    monkeypatch.setattr("sys.argv", ["decoder_layer.py", "--tokens", "6", "--seqs", "3", "--prompt", "100", "--budget", "64", "--shape", "512", "4", "2", "768"])
    ex.main()
    assert "us a step" in capsys.readouterr().out


def test_example_runs_past_the_layers_usual_positions(gpu, monkeypatch, capsys):
    ex = _example()
    monkeypatch.setattr("sys.argv", ["decoder_layer.py", "--tokens", "3", "--seqs", "2", "--prompt", "4095", "--budget", "100", "--shape", "256", "4", "2", "512"])
    ex.main()
    assert "us a step" in capsys.readouterr().out
