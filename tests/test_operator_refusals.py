"""What the operators refuse, before any launch (no GPU needed)."""
import ctypes

import pytest
import torch

import dlcompiler_b200 as dl
from dlcompiler_b200 import _lib


@pytest.fixture()
def no_launch(monkeypatch):
    """CPU tensors pass for CUDA ones, and getting as far as the library is a failure."""
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "load", lambda: pytest.fail("not refused"))


def test_cpu_tensors_are_refused():
    t = torch.zeros(2, 2, 16)
    with pytest.raises(AssertionError, match="CUDA"):
        dl.apply_multi_axis_rotary(t, t, torch.zeros(1, 2, dtype=torch.int64), torch.ones(8), [8])


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(6, 32)), dict(k=torch.zeros(3, 1, 16)), dict(k=torch.zeros(2, 1, 24)),
    dict(k=torch.zeros(2, 1, 16).half()), dict(positions=torch.zeros(2, dtype=torch.int64)),
    dict(positions=torch.zeros(2, 3, dtype=torch.int64)), dict(positions=torch.zeros(2, 2)),
    dict(inv_freq=torch.ones(8).double()), dict(inv_freq=torch.ones(2, 4)), dict(inv_freq=torch.ones(8).requires_grad_()),
    dict(sections=[8]), dict(sections=[4, 5]), dict(sections=[9, -1]),
    dict(q_embed=torch.zeros(2, 3, 8)), dict(q_embed=torch.zeros(2, 3, 16).half()),
    dict(k_embed=torch.zeros(2, 16, 1).transpose(1, 2).expand(2, 1, 16)[..., ::1].repeat(1, 1, 2)[..., ::2]),
    dict(q=torch.zeros(2, 3, 16).requires_grad_(), q_embed=torch.zeros(2, 3, 16)),
])
def test_multi_axis_rotary(no_launch, change):
    args = dict(q=torch.zeros(2, 3, 16), k=torch.zeros(2, 1, 16), positions=torch.zeros(2, 2, dtype=torch.int64),
                inv_freq=torch.ones(8), sections=[4, 4])
    args.update(change)
    with pytest.raises(AssertionError):
        dl.apply_multi_axis_rotary(**args)


def test_multi_axis_rotary_entry():
    lib = _lib.load()
    axes = (ctypes.c_uint8 * 300)(*([0, 1] * 150))

    def call(q=16, axis_map=axes, n_axes=2, tokens=4, dim=64, rot=64, dtype=_lib.DTYPE_BF16):
        return lib.dlb_multi_axis_rotary(q, 16, 16, 16, 16, 1, 4, 16, axis_map, n_axes, tokens, 2, 1, dim, rot,
                                         128, 64, 64, 64, 128, 64, 64, 64, 0, dtype, None)

    for bad in (dict(q=None), dict(axis_map=None), dict(n_axes=0), dict(n_axes=9), dict(n_axes=1), dict(tokens=-1),
                dict(tokens=1 << 31), dict(rot=63), dict(rot=66), dict(rot=0), dict(dim=600, rot=520), dict(dtype=7)):
        assert call(**bad) < 0 and lib.dlb_last_error().startswith(b"multi_axis_rotary"), bad
    assert call(tokens=0) == 0
