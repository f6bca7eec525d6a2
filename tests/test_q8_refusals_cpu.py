"""More of what the operators of the 8-bit cache and of the step's maps refuse, and how their front chooses, without a GPU."""

from types import SimpleNamespace

import pytest
import torch

from tests.test_q8_cache_cpu import I32, attend_args, ops  # noqa: F401


def step(**other):
    a = dict(num_requests=3, num_decode=3, q_start=torch.arange(4, dtype=I32), seq_lens=torch.ones(3, dtype=I32), max_q_len=1, max_seq_len=1)
    a.update(other)
    return SimpleNamespace(**a)


@pytest.mark.parametrize("other", [
    dict(q_start=torch.arange(4)), dict(q_start=torch.arange(4.0)), dict(q_start=torch.arange(3, dtype=I32)),
    dict(q_start=torch.arange(8, dtype=I32)[::2]), dict(q_start=torch.zeros(4, 1, dtype=I32)),
    dict(seq_lens=torch.ones(3, dtype=torch.int64)), dict(seq_lens=torch.ones(2, dtype=I32)), dict(seq_lens=torch.ones(6, dtype=I32)[::2]),
    dict(seq_lens=torch.ones(1, 3, dtype=I32)), dict(num_decode=4), dict(num_decode=-1),
], ids=lambda o: "-".join(f"{k}{tuple(v.shape)}{v.dtype}" if isinstance(v, torch.Tensor) else f"{k}{v}" for k, v in o.items()))
def test_attention_refuses_a_step_that_does_not_fit(ops, other):  # noqa: F811
    with pytest.raises(ValueError, match="query starts"):
        ops.attention_q8(**attend_args(step=step(**other)))


class Elsewhere(torch.Tensor):
    def get_device(self):
        return 1


@pytest.mark.parametrize("which", ["q_start", "seq_lens"])
def test_attention_refuses_a_step_of_another_device(ops, which):  # noqa: F811
    """Everything on the kernels' device (the CPU's number here) but one of the step's arrays."""
    with pytest.raises(ValueError, match="must be on GPU"):
        ops.attention_q8(**attend_args(step=step(**{which: getattr(step(), which).as_subclass(Elsewhere)})))


def test_portions_where_the_device_does_not_hold_a_block_are_left_to_the_kernel_for_any_sizes():
    """The tensor cores' kernel answers "not taken by this kernel", upon which the front calls the other one: on a machine without a GPU it
    cannot be configured."""
    import ctypes
    import os

    from turingserve_b200 import kernels
    from turingserve_b200.kernels import _ATTEND_Q8, CudaOps

    if torch.cuda.is_available():
        pytest.skip("this machine's GPU holds the kernel")
    path = os.path.join(os.path.dirname(kernels.__file__), "libturingserve_b200.so")
    if not os.path.exists(path):
        pytest.skip("the library is not built")
    lib = ctypes.CDLL(path)
    lib.ts_attention_q8_prefill.argtypes = [ctypes.c_char_p, ctypes.c_void_p]
    for D in (64, 128):
        page = torch.zeros(64 * 128 * 2, dtype=torch.uint8)
        at = page.data_ptr() // 16 * 16 + 16
        record = _ATTEND_Q8.pack(*(at,) * 6, at, at, at, 0, D, D, 1, 1, 16, 16, 1, 1, D, 16, 1, 0, 1, 1, 0, 0, 0.1)
        assert lib.ts_attention_q8_prefill(record, None) == CudaOps.UNSUPPORTED


class Recorder:
    """A library whose single tokens' kernel notes what it is called with; clusters may be switched off behind the front's back."""

    def __init__(self):
        self.clusters, self.calls = True, []

    def ts_attention_q8_decode_blocks_per_sm(self, G, D):
        return 2

    def ts_attention_q8_decode_clusters(self, G, D, n):
        return 100

    def ts_attention_q8_decode(self, record, stream):
        from turingserve_b200.kernels import _ATTEND_Q8
        fields = _ATTEND_Q8.unpack(record)
        scratch, splits, cluster = fields[9], fields[-4], fields[-3]
        self.calls.append((splits, bool(cluster), scratch != 0))
        return -4 if cluster and not self.clusters else 0


def test_clusters_switched_off_after_the_first_call(ops, monkeypatch):  # noqa: F811
    """And on again: the choice between a cluster and scratch is the call's, not the first call's."""
    ops.lib, ops._q8_plans, ops.launches, ops.use_fast_attention = Recorder(), {}, 0, True
    monkeypatch.setattr(ops, "_stream", lambda: 0, raising=False)
    args = attend_args(step=step(max_seq_len=600))
    launches = []
    for on in (True, False, True):
        ops.lib.clusters = on
        before = ops.launches
        ops.attention_q8(**args)
        launches.append(ops.launches - before)
        splits, cluster, scratch = ops.lib.calls[-1]
        assert splits > 1 and cluster == on and scratch == (not on)
    assert launches == [1, 2, 1]
