"""The serving example against the same layer in 64 bits, a talk at a time."""
import importlib.util
from pathlib import Path

import numpy as np
import pytest

from onnx_runtime_dart_amd import _lib
from oracle import refcpu
from tests.paged_cases import to_type

pytestmark = pytest.mark.gpu
PATH = Path(__file__).resolve().parents[1] / "examples" / "paged_serving.py"


def load():
    spec = importlib.util.spec_from_file_location("paged_serving", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def weights(w, k, n, block=32):
    """[k, n] in 64 bits of packed int4 weights: the product with unit rows."""
    b, s, z = w
    return refcpu.matmul_nbits(np.eye(k, dtype=np.float32), b, s, z, k, n, 4,
                               block).astype(np.float64)


def reference(layer, system, prompts, given, t):
    """Every talk alone over system + its rows; `given` are the rows that the device fed back."""
    H, G, D = layer.heads, layer.kv_heads, layer.head
    wq = weights(layer.weights[0], layer.hidden, layer.width)
    wo = weights(layer.weights[1], H * D, layer.hidden)
    cos, sin = (x.astype(np.float64) for x in layer.tables)
    out = []
    for prompt, rows in zip(prompts, given):
        # a step's input is the result before it
        x = np.concatenate([system, prompt, rows[len(prompt) - 1:-1]]).astype(np.float64)
        y = (x @ wq).reshape(len(x), H + 2 * G, D)
        turn = y[:, :H + G].copy()
        c, s = cos[:len(x), None], sin[:len(x), None]
        half = layer.half
        turn[..., :half] = y[:, :H + G, :half] * c - y[:, :H + G, half:] * s
        turn[..., half:] = y[:, :H + G, half:] * c + y[:, :H + G, :half] * s
        k, v = (to_type(z, t)[1] for z in (turn[:, H:], y[:, H + G:]))
        seen = np.tril(np.ones((len(x), len(x)), bool))
        o = np.empty((len(x), H, D))
        for h in range(H):
            z = np.where(seen, turn[:, h] @ k[:, h // (H // G)].T / np.sqrt(D), -np.inf)
            e = np.exp(z - z.max(-1, keepdims=True))
            o[:, h] = e / e.sum(-1, keepdims=True) @ v[:, h // (H // G)]
        out.append((o.reshape(len(x), H * D) @ wo + x)[len(system):])
    return out


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
def test_serving_example(t):
    """A cached value that the device computes on the other side of a rounding border differs
    by a whole step of its type (twice the half step that both sides round by), and so may
    the attention of which it is a part; the projections and sums before and after add
    binary32's roundings, 2^-24 each, over sums of 512 terms and softmax weights: 2^-17."""
    mod = load()
    layer = mod.Layer(_lib.default_context(), dtype=t, max_pos=512, seed=3)
    rng = np.random.default_rng(7)
    system = rng.standard_normal((90, layer.hidden)).astype(np.float32)
    prompts = [rng.standard_normal((m, layer.hidden)).astype(np.float32) for m in (1, 40, 17, 65)]
    got = mod.serve(layer, system, prompts, 6)
    want = reference(layer, system, prompts, got, t)
    step = {"f32": 0.0, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}[t]
    for y, w, p in zip(got, want, prompts):
        assert y.shape == (len(p) + 6, layer.hidden)
        off = np.abs(y - w).max() / np.abs(w).max()
        print(f"{len(p)} rows: {off:.3g} of the largest value", flush=True)
        assert off <= 2.0 ** -17 + step
