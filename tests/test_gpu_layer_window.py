"""GPU: decoder blocks whose attention has a sliding window and sinks
(BlockConfig.window, .sinks) against the oracle's block around plain attention in
64 bits with the same mask: prompts, single tokens, a recorded step."""
import dataclasses

import numpy as np
import pytest

import paged_ref as R
import test_gpu_layer as L
from conftest import RTOL, rel_to_scale
from aero_amd import layer
from aero_amd import workloads as W
from aero_amd.device import Plan

pytestmark = pytest.mark.gpu


class Windowed:
    """The oracle with the block's attention in 64 bits under a window and sinks."""

    def __init__(self, oracle, window, sinks):
        self.oracle, self.window, self.sinks = oracle, window, sinks

    def __getattr__(self, name):
        return getattr(self.oracle, name)

    def attention_tiled(self, q, k, v, scale, qpos=None, kpos=None):
        return R.attention(q, k, v, R.seen(qpos, kpos, self.window, self.sinks),
                           scale).astype(np.float32)


def block(shape, T, kv_len, window, sinks):
    cfg = layer.BlockConfig.from_shape(W.SHAPES[shape], W.Q8_0, vocab=2048, window=window,
                                       sinks=sinks)
    wts = layer.BlockWeights(cfg, seed=3)
    step = layer.LayerStep(cfg, wts, max_tokens=T, kv_cap=kv_len + T)
    rng = np.random.default_rng(4)
    ids = rng.integers(0, cfg.vocab, T).astype(np.int32)
    K0, V0 = (rng.standard_normal((kv_len + T, cfg.n_head_kv * cfg.head_dim), dtype=np.float32)
              for _ in range(2))
    for dev, host in zip(step.kv[0], (K0, V0)):
        dev.copy_from(host)
    return cfg, wts, step, ids, K0, V0


@pytest.mark.parametrize("shape,T,kv_len,window,sinks", [
    ("qwen2_0p5b_decode", 1, 200, 64, 4), ("qwen2_0p5b_decode", 1, 200, 64, 0),
    ("qwen2_0p5b_decode", 40, 100, 33, 16), ("llama3_8b_prefill", 520, 70, 100, 4),
    ("gemma3_4b_prefill", 48, 30, 20, 1)])
def test_block_with_window(hip, oracle, shape, T, kv_len, window, sinks):
    cfg, wts, step, ids, K0, V0 = block(shape, T, kv_len, window, sinks)
    step.prepare(ids, kv_len)
    step.forward(T, kv_len)
    want_x, want_h = L.oracle_block(Windowed(oracle, window, sinks), cfg, wts, ids, kv_len, K0, V0)
    assert rel_to_scale(step.x.view((T, cfg.hidden)).numpy(), want_x) <= RTOL
    assert rel_to_scale(step.h_out.view((T, cfg.hidden)).numpy(), want_h) <= RTOL
    # the mask matters: without it the block's result is another one
    plain = dataclasses.replace(cfg, window=0, sinks=0)
    other, _ = L.oracle_block(oracle, plain, wts, ids, kv_len, K0, V0)
    assert rel_to_scale(other, want_x) > 10 * RTOL


def test_recorded_block_with_window(hip, oracle):
    """Recorded once, replayed over the cache as the step before left it."""
    kv_len, window, sinks = 90, 32, 4
    cfg, wts, step, ids, K0, V0 = block("qwen2_0p5b_decode", 1, kv_len, window, sinks)
    step.prepare(ids, kv_len)
    plan = Plan()
    with plan:
        step.forward(1, kv_len)
    want_x, want_h = L.oracle_block(Windowed(oracle, window, sinks), cfg, wts, ids, kv_len, K0, V0)
    for _ in range(3):
        plan.launch()
        assert rel_to_scale(step.x.view((1, cfg.hidden)).numpy(), want_x) <= RTOL
        assert rel_to_scale(step.h_out.view((1, cfg.hidden)).numpy(), want_h) <= RTOL
    plan.destroy()
