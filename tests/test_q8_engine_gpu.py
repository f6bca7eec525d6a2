"""The engine with its cache in 8 bits: steps against a plain model whose cache is the 64-bit one of ``plain_q8``, generation through the
public entry points, portions, preemption, captured steps, other layers' caches.

How near.  The float32 engine works the plain model's formulas in 32 bits; where a key or value lies within that rounding of a border
between two 8-bit values (about one in 2^17 at errors of 2^-21) it may be held as the neighbour.  So its logits differ from the
plain ones by what a few of some ten thousand values moved by one step do, while leaving the rounding out altogether moves every one of them by
up to half a step: the square root of a few in ten thousand, far below a quarter of that distance, is what is asked.  The bfloat16 engine rounds
every activation to 2^-8 besides: its tokens are the best ones within 5 % of the largest logit, as for the engine's other caches."""

from __future__ import annotations

import pytest
import torch

from tests import plain_q8, tiny
from tests import plain_qwen2 as plain
from tests.test_engine_gpu import engine, greedy, tokens_are_best

pytestmark = pytest.mark.gpu


class PlainQ8:
    """A plain model of one sequence, step by step, its cache in pages of 8 bits (float32 products, 64-bit cache and attention)."""

    def __init__(self, cfg, w, page, dtype=torch.float32):
        self.cfg, self.w, self.s, self.page, self.n = cfg, w, plain.sizes(cfg), page, 0
        self.dtype = dtype
        pages = 64
        shape = (pages, self.s["KVH"], page, self.s["D"])
        self.caches = [[torch.zeros(shape, dtype=torch.float64), torch.ones(shape[:2], dtype=torch.float64)] for _ in range(2 * self.s["L"])]
        self.table = torch.arange(pages, dtype=torch.int32)[None]

    @torch.inference_mode()
    def step(self, tokens):
        s, w, cfg = self.s, self.w, self.cfg
        T = len(tokens)
        pos = torch.arange(self.n, self.n + T)
        cos, sin = plain.rope_tables(s["D"], s["theta"], self.n + T)
        h, residual = w["model.embed_tokens.weight"][torch.tensor(tokens)], None
        for layer in range(s["L"]):
            p = f"model.layers.{layer}."
            residual = h if residual is None else h + residual
            x = plain.rmsnorm(residual, w[p + "input_layernorm.weight"], s["eps"])
            q, k, v = plain.qkv_projection(x, w, p, s)
            q = plain.apply_rope(q, pos, cos, sin)
            k = plain_q8.rotate(k.double(), pos, cos, sin, s["D"], self.dtype)
            (kc, ks), (vc, vs) = self.caches[2 * layer], self.caches[2 * layer + 1]
            plain_q8.write_rows(kc, ks, k, pos.tolist())
            plain_q8.write_rows(vc, vs, v.double(), pos.tolist())
            a, _, _ = plain_q8.attend(q, kc, vc, ks, vs, self.table, [T], [self.n + T], self.page, s["D"] ** -0.5, plain.layer_window(cfg, layer))
            h = torch.nn.functional.linear(a.float().reshape(T, -1), w[p + "self_attn.o_proj.weight"])
            residual = h + residual
            x = plain.rmsnorm(residual, w[p + "post_attention_layernorm.weight"], s["eps"])
            h = plain.mlp(x, w[p + "mlp.gate_proj.weight"], w[p + "mlp.up_proj.weight"], w[p + "mlp.down_proj.weight"])
        self.n += T
        x = plain.rmsnorm(h + residual, w["model.norm.weight"], s["eps"])
        head = w["model.embed_tokens.weight"] if s["tied"] else w["lm_head.weight"]
        return torch.nn.functional.linear(x, head).float()


def q8_engine(folder, dtype="float32", **kw):
    return engine(folder, dtype, kv_cache_dtype="fp8", **kw)


@pytest.mark.parametrize("name", ["A", "B", "W", "K", "L", "X"])
def test_steps_float32(tmp_path, name):
    folder = tiny.make_tiny_folder(name, tmp_path)
    cfg, w = plain.read_folder(folder)
    eng = q8_engine(folder, block_size=16)
    from turingserve_b200.engine.batch import StepEntry
    ids = tiny.random_ids(80, cfg["vocab_size"], 3)
    cuts = [33, 20, 1, 1, 9, 1, 1]
    rc, model, at, got, want = eng.cache.admit("r"), PlainQ8(cfg, w, 16), 0, [], []
    for n in cuts:
        got.append(eng.runner.step([StepEntry(rc, ids[at:at + n], list(range(n)))]).float().cpu())
        want.append(model.step(ids[at:at + n]))
        at += n
    got, want = torch.cat(got), torch.cat(want)
    whole = plain.forward(cfg, w, ids[:at])
    off, rounding = (got - want).norm(), (whole - want).norm()
    assert float(rounding) > 0 and float(off) < 0.25 * float(rounding), (float(off), float(rounding))


@pytest.mark.parametrize("name,block", [("K", 16), ("K", 64), ("L", 32)])
@pytest.mark.parametrize("graphs", [True, False])
def test_generation_bfloat16(tmp_path, name, block, graphs):
    folder = tiny.make_tiny_folder(name, tmp_path)
    cfg, w = plain.read_folder(folder)
    prompts = [tiny.random_ids(n, cfg["vocab_size"], 20 + n) for n in (5, 17, 130, 1, 64)]
    eng = q8_engine(folder, "bfloat16", block_size=block, max_num_batched_tokens=64, cuda_graphs=graphs)
    outs = eng.generate(prompts, greedy(12))
    for p, o in zip(prompts, outs):
        tokens_are_best(cfg, w, p, o.token_ids, 0.05)
        assert len(o.token_ids) == 12
    assert not eng.faults and eng.cache.min_free() == eng.cache.num_pages - 1
    eng.cache.check()


def test_preemption_and_pages_that_are_used_again(tmp_path):
    """Few pages: requests are thrown out and come back, pages go from hand to hand with the scales of their last owner in them."""
    folder = tiny.make_tiny_folder("K", tmp_path)
    cfg, w = plain.read_folder(folder)
    prompts = [tiny.random_ids(n, cfg["vocab_size"], 40 + n) for n in (30, 41, 25, 50, 33, 28)]
    eng = q8_engine(folder, "bfloat16", num_blocks=14, max_num_seqs=6, max_num_batched_tokens=48)
    outs = eng.generate(prompts, greedy(24))
    for p, o in zip(prompts, outs):
        tokens_are_best(cfg, w, p, o.token_ids, 0.05)
        assert len(o.token_ids) == 24
    eng.cache.check()


def test_twice_as_many_pages_in_the_same_memory(tmp_path):
    from turingserve_b200.cache.manager import CacheManager
    from turingserve_b200.engine.runner import run_needs
    folder = tiny.make_tiny_folder("K", tmp_path)
    eng = q8_engine(folder, "bfloat16")
    needs = run_needs(eng.runner.model)
    assert eng.runner.fused is None                              # the one-kernel step reads bfloat16 caches
    wide, narrow = (CacheManager.bytes_per_page(needs, 64, t) for t in (torch.bfloat16, torch.float8_e4m3fn))
    assert narrow * 2 - wide == 2 * 8 * 2 * 2                    # (the scales: 8 bytes a kv head, two layers of two)
    group = eng.cache.groups[0]
    assert group.pool.dtype == torch.float8_e4m3fn and group.scales.shape == (2, 2, eng.cache.num_pages, 2)


def test_a_product_that_is_not_finished(tmp_path):
    """The write sums a split product itself: the same pages as from the finished product."""
    from turingserve_b200 import kernels
    kernels.use(None)
    ops = kernels.ops()
    g = torch.Generator(device="cuda").manual_seed(4)
    for T, H, KVH, D, splits in ((1, 12, 2, 128, 3), (8, 14, 2, 64, 1), (40, 28, 4, 128, 8), (100, 4, 4, 64, 16)):
        n, page = (H + 2 * KVH) * D, 16
        part = torch.randn((splits, T, n), generator=g, device="cuda")
        for bias in (None, torch.randn(n, generator=g, device="cuda").bfloat16()):
            whole = torch.zeros((T, n), device="cuda")
            for s in range(splits):
                whole += part[s]
            whole = (whole if bias is None else whole + bias.float()).bfloat16()
            freq = 10000.0 ** (-torch.arange(0, D, 2, device="cuda").double() / D)
            angle = torch.arange(200, device="cuda").double()[:, None] * freq
            cos, sin = angle.cos().float(), angle.sin().float()
            pos = torch.arange(50, 50 + T, device="cuda").int()
            outs = []
            for x in (whole, kernels.Deferred(part, splits, (T, n), torch.bfloat16, bias, torch.empty_like(whole))):
                k = torch.zeros((20, KVH, page, D), dtype=torch.float8_e4m3fn, device="cuda")
                v, ks = torch.zeros_like(k), torch.ones((20, KVH), device="cuda")
                vs, q = torch.ones_like(ks), torch.empty((T, H * D), dtype=torch.bfloat16, device="cuda")
                ops.rope_kv_write_q8(q, x, pos, cos, sin, H, KVH, D, D, k, v, ks, vs, pos, page)
                outs.append((q, k.view(torch.uint8), v.view(torch.uint8), ks, vs))
            assert all(torch.equal(a, b) for a, b in zip(*outs))
