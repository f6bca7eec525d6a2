"""What the operators of the 8-bit cache and of the step's maps refuse, before anything reaches the GPU; and the plain forms themselves."""

from types import SimpleNamespace

import math

import pytest
import torch

from tests import plain_q8 as plain
from turingserve_b200.kernels import CudaOps

F8, BF16, I32 = torch.float8_e4m3fn, torch.bfloat16, torch.int32


class NoLibrary:
    def __getattr__(self, name):
        raise AssertionError(f"{name} was called")


@pytest.fixture
def ops():
    o = CudaOps.__new__(CudaOps)
    o.lib, o.num_sms, o._device_index = NoLibrary(), 148, -1      # (-1: the CPU's, so that only what is wrong refuses)
    return o


def write_args(T=3, H=4, KVH=2, D=64, page=16, **other):
    a = dict(q_out=torch.zeros(T, H * D, dtype=BF16), qkv=torch.zeros(T, (H + 2 * KVH) * D, dtype=BF16), positions=torch.zeros(T, dtype=I32),
             cos=torch.zeros(8, D // 2), sin=torch.zeros(8, D // 2), H=H, KVH=KVH, D=D, rotary_dim=D,
             k_cache=torch.zeros(5, KVH, page, D, dtype=F8), v_cache=torch.zeros(5, KVH, page, D, dtype=F8), k_scale=torch.ones(5, KVH),
             v_scale=torch.ones(5, KVH), slots=torch.zeros(T, dtype=I32), page_size=page)
    a.update(other)
    return a


@pytest.mark.parametrize("other", [
    dict(qkv=torch.zeros(3, 500, dtype=BF16)),
    dict(qkv=torch.zeros(3, 1024, dtype=BF16)[:, ::2]),
    dict(qkv=torch.zeros(3, 512, dtype=torch.float32)),
    dict(q_out=torch.zeros(2, 256, dtype=BF16)),
    dict(q_out=torch.zeros(256, 3, dtype=BF16).t()),
    dict(positions=torch.zeros(3, dtype=torch.int64)),
    dict(positions=torch.zeros(4, dtype=I32)),
    dict(positions=torch.zeros(6, dtype=I32)[::2]),
    dict(slots=torch.zeros(3, dtype=torch.int64)),
    dict(slots=torch.zeros(6, dtype=I32)[::2]),
    dict(k_cache=torch.zeros(5, 2, 16, 64, dtype=BF16)),
    dict(v_cache=torch.zeros(5, 2, 16, 64, dtype=torch.uint8)),
    dict(v_cache=torch.zeros(4, 2, 16, 64, dtype=F8)),
    dict(k_cache=torch.zeros(5, 2, 8, 64, dtype=F8)),
    dict(k_cache=torch.zeros(5, 16, 2, 64, dtype=F8).transpose(1, 2)),
    dict(k_scale=torch.ones(5, 2, dtype=torch.float64)),
    dict(v_scale=torch.ones(5, 3)),
    dict(v_scale=torch.ones(2, 5).t()),
    dict(rotary_dim=65), dict(rotary_dim=66), dict(rotary_dim=-2),
    dict(cos=None), dict(sin=torch.zeros(8, 32, dtype=BF16)), dict(sin=torch.zeros(8, 16)), dict(cos=torch.zeros(8, 64)[:, ::2]),
    dict(slots=None), dict(v_cache=None), dict(k_scale=None),
])
def test_write_refuses(ops, other):
    with pytest.raises((ValueError, TypeError)):
        ops.rope_kv_write_q8(**write_args(**other))


def attend_args(**other):
    a = dict(out=torch.zeros(3, 256, dtype=BF16), q=torch.zeros(3, 4, 64, dtype=BF16), k_cache=torch.zeros(5, 2, 16, 64, dtype=F8),
             v_cache=torch.zeros(5, 2, 16, 64, dtype=F8), k_scale=torch.ones(5, 2), v_scale=torch.ones(5, 2),
             block_tables=torch.zeros(3, 4, dtype=I32),
             step=SimpleNamespace(num_requests=3, num_decode=3, q_start=torch.arange(4, dtype=I32), seq_lens=torch.ones(3, dtype=I32),
                                  max_q_len=1, max_seq_len=1),
             KVH=2, page_size=16, scale=0.1, window=None)
    a.update(other)
    return a


@pytest.mark.parametrize("other", [
    dict(q=torch.zeros(3, 5, 64, dtype=BF16)),
    dict(q=torch.zeros(3, 64, 4, dtype=BF16).transpose(1, 2)),
    dict(q=torch.zeros(3, 4, 64, dtype=torch.float16), out=torch.zeros(3, 256, dtype=torch.float16)),
    dict(out=torch.zeros(3, 256)),
    dict(out=torch.zeros(3, 4, 64, dtype=BF16)),
    dict(out=torch.zeros(2, 256, dtype=BF16)),
    dict(k_cache=torch.zeros(5, 2, 16, 64, dtype=BF16)),
    dict(v_cache=torch.zeros(5, 2, 16, 128, dtype=F8)),
    dict(v_scale=torch.ones(5, 2, 1)),
    dict(block_tables=torch.zeros(3, 4, dtype=torch.int64)),
    dict(block_tables=torch.zeros(2, 4, dtype=I32)),
    dict(block_tables=torch.zeros(4, 3, dtype=I32).t()),
    dict(window=-1),
])
def test_attention_refuses(ops, other):
    with pytest.raises((ValueError, TypeError)):
        ops.attention_q8(**attend_args(**other))


def maps_args(**other):
    z = lambda *s: torch.zeros(s, dtype=I32)  # noqa: E731
    a = dict(requests=z(3, 2), updates=z(1, 4), tables=z(2, 5, 7), page_size=16, q_start=z(3), seq_lens=z(2), token_request=z(4),
             positions=z(4), slot_mapping=z(2, 4), block_tables=z(2, 2, 7))
    a.update(other)
    return a


@pytest.mark.parametrize("other", [
    dict(requests=torch.zeros(2, 2, dtype=I32)), dict(requests=torch.zeros(3, 2, dtype=torch.int64)),
    dict(requests=torch.zeros(2, 3, dtype=I32).t()), dict(updates=torch.zeros(1, 3, dtype=I32)), dict(updates=torch.zeros(4, dtype=I32)),
    dict(tables=torch.zeros(5, 7, dtype=I32)), dict(q_start=torch.zeros(2, dtype=I32)), dict(seq_lens=torch.zeros(3, dtype=I32)),
    dict(token_request=torch.zeros(3, dtype=I32)), dict(positions=torch.zeros(4, 1, dtype=I32)), dict(slot_mapping=torch.zeros(1, 4, dtype=I32)),
    dict(block_tables=torch.zeros(2, 3, 7, dtype=I32)), dict(block_tables=torch.zeros(2, 7, dtype=I32)), dict(page_size=0),
])
def test_maps_refuse(ops, other):
    with pytest.raises(ValueError):
        ops.step_maps(**maps_args(**other))


def test_tensors_of_another_device_are_refused(ops):
    ops._device_index = 0
    for call, args in ((ops.rope_kv_write_q8, write_args()), (ops.rope_kv_write_q8, write_args(k_cache=None)), (ops.attention_q8, attend_args()),
                       (ops.step_maps, maps_args())):
        with pytest.raises(ValueError, match="on GPU 0"):
            call(**args)


def test_scales():
    for top, want in ((448.0, 1.0), (448.0 * (1 + 2 ** -20), 2.0), (449.0, 2.0), (224.0, 0.5), (224.1, 1.0), (1.0, 2.0 ** -8), (0.0, 2.0 ** -50),
                      (2.0 ** -70, 2.0 ** -50), (448.0 * 2.0 ** 50, 2.0 ** 50)):
        assert plain.scale_for(top) == want
    for top in (math.inf, math.nan, 450.0 * 2.0 ** 50):
        assert math.isnan(plain.scale_for(top))


def test_rounding_is_torchs():
    x = torch.cat([torch.randn(4000, dtype=torch.float64, generator=torch.Generator().manual_seed(0)) * s for s in (200.0, 1.0, 0.01, 0.002)])
    x = x.clamp(-448, 448).float()
    assert torch.equal(plain.e4m3(x.double()), x.to(F8).double())


# -- the engine's side, without a GPU ---------------------------------------------------------------------------------------

def test_engine_option():
    from turingserve_b200 import EngineConfig
    from turingserve_b200.config.engine_config import add_engine_arguments, engine_config_from_namespace
    import argparse

    assert EngineConfig(model="x").torch_cache_dtype is BF16
    assert EngineConfig(model="x", dtype="float32").torch_cache_dtype is torch.float32
    assert EngineConfig(model="x", dtype="float32", kv_cache_dtype="fp8").torch_cache_dtype is F8
    with pytest.raises(ValueError, match="kv-cache-dtype"):
        EngineConfig(model="x", kv_cache_dtype="int8").validate()
    p = argparse.ArgumentParser()
    add_engine_arguments(p)
    assert engine_config_from_namespace(p.parse_args(["--model", "x", "--kv-cache-dtype", "fp8"])).kv_cache_dtype == "fp8"
    assert engine_config_from_namespace(p.parse_args(["--model", "x"])).kv_cache_dtype == "auto"


def test_cache_manager_in_8_bits():
    from turingserve_b200.cache import CacheManager, RunNeeds
    from turingserve_b200.parts.base import CacheNeed
    needs = [RunNeeds(CacheNeed(2, 8), None), RunNeeds(CacheNeed(2, 8, 16), None), RunNeeds(CacheNeed(2, 8), None), RunNeeds(None, None, 0)]
    m = CacheManager(needs, 4, 6, 3, F8, "cpu")
    v = m.views()
    assert v[0].k.dtype == F8 and v[0].k.shape == (6, 2, 4, 8) and v[2].v_scale.shape == (6, 2) and v[1].k_scale.shape == (6, 2)
    assert v[0].k_scale.data_ptr() != v[2].k_scale.data_ptr() != v[2].v_scale.data_ptr()
    assert v[3].k_scale.data_ptr() == v[0].k_scale.data_ptr() and not v[3].writable
    assert all(x.k_scale.is_contiguous() and x.k_scale.eq(1).all() for x in v)
    assert CacheManager(needs, 4, 6, 3, BF16, "cpu").views()[0].k_scale is None
    with pytest.raises(ValueError, match="one width"):
        CacheManager([RunNeeds(CacheNeed(1, 8, value_dim=4), None)], 4, 6, 3, F8, "cpu")
    a, b = m.admit("a"), m.admit("b")
    m.release(a)
    assert b.admission != a.admission != m.admit("c").admission


def test_models_whose_mixers_keep_the_engines_type_are_refused():
    from turingserve_b200.engine.runner import check_cache_dtype

    class Mixer:
        def __init__(self, need, takes):
            self.takes_q8_cache, self._need = takes, need

        def cache_need(self):
            return self._need
    make = lambda *mixers: SimpleNamespace(cfg=SimpleNamespace(schedule=range(len(mixers))), run_mixer=lambda r: mixers[r])  # noqa: E731
    check_cache_dtype(make(Mixer(1, True), Mixer(None, False)), F8)
    check_cache_dtype(make(Mixer(1, False)), BF16)
    with pytest.raises(ValueError, match="Mixer"):
        check_cache_dtype(make(Mixer(1, True), Mixer(1, False)), F8)
