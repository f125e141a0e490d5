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


def _attention_args(tokens=3):
    cache = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    q = torch.zeros(tokens, 4, 64, dtype=torch.bfloat16)
    lens = torch.ones(3, dtype=torch.int32)
    return dict(q=q, k=cache, v=cache.clone(), o=q.clone(), block_offsets=torch.zeros(3, 2, dtype=torch.int32), kv_seqlens=lens)


SHARED = [
    dict(q=torch.zeros(3, 256, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 4, 64)),
    dict(q=torch.zeros(3, 4, 64, dtype=torch.float16)), dict(q=torch.zeros(3, 3, 64, dtype=torch.bfloat16)),
    dict(q=torch.zeros(3, 4, 32, dtype=torch.bfloat16)), dict(q=torch.zeros(3, 258, 64, dtype=torch.bfloat16)),
    dict(k=torch.zeros(64, 2, 64, dtype=torch.bfloat16)), dict(k=torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)[..., ::2]),
    dict(v=torch.zeros(4, 16, 1, 64, dtype=torch.bfloat16)), dict(v=torch.zeros(4, 16, 2, 64)),
    dict(v=torch.zeros(4, 16, 2, 32, dtype=torch.bfloat16)), dict(o=torch.zeros(2, 4, 64, dtype=torch.bfloat16)),
    dict(o=torch.zeros(3, 64, 4, dtype=torch.bfloat16).transpose(1, 2)), dict(o=torch.zeros(3, 4, 64)),
    dict(block_offsets=torch.zeros(2, 2, dtype=torch.int32)), dict(block_offsets=torch.zeros(3, 0, dtype=torch.int32)),
    dict(block_offsets=torch.zeros(3, dtype=torch.int32)), dict(kv_seqlens=torch.ones(2, dtype=torch.int32)),
]


@pytest.mark.parametrize("change", SHARED + [
    dict(q_start_loc=torch.zeros(2, dtype=torch.int32)), dict(window_size=-1), dict(num_sinks=-1), dict(max_seqlen=-1)])
def test_sink_attention(no_launch, change):
    args = _attention_args()
    args.update(q_start_loc=torch.arange(3), q_seqlens=torch.ones(3, dtype=torch.int32), max_seqlen=1, window_size=8, num_sinks=2)
    args.update(change)
    with pytest.raises(AssertionError):
        dl.sink_attention_fwd(**args)


@pytest.mark.parametrize("change", SHARED + [
    dict(prefix_offsets=torch.zeros(2, dtype=torch.int32)), dict(prefix_offsets=torch.zeros(1, 2, dtype=torch.int32)),
    dict(prefix_offsets=torch.zeros(2, 0, dtype=torch.int32)), dict(group_start=torch.zeros(2, dtype=torch.int32)),
    dict(prefix_seqlens=torch.zeros(0, dtype=torch.int32), group_start=torch.zeros(1, dtype=torch.int32))])
def test_shared_prefix_attention(no_launch, change):
    args = _attention_args()
    args.update(prefix_offsets=torch.zeros(2, 2, dtype=torch.int32), prefix_seqlens=torch.ones(2, dtype=torch.int32),
                group_start=torch.tensor([0, 1, 3], dtype=torch.int32))
    args.update(change)
    with pytest.raises(AssertionError):
        dl.shared_prefix_attention_fwd(**args)


@pytest.mark.parametrize("name", ["block_offsets", "q_start_loc", "q_seqlens", "kv_seqlens"])
def test_sink_attention_index_types(monkeypatch, name):
    """Any library call is a failure: the index tensors are looked at first."""
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: torch.device("cpu", 0))
    monkeypatch.setattr(_lib, "on_device", lambda d: _lib._CURRENT_DEVICE)
    monkeypatch.setattr(_lib, "stream_ptr", lambda d: 0)

    class Lib:
        def __getattr__(self, entry):
            return lambda *a: pytest.fail("not refused")

    monkeypatch.setattr(_lib, "load", Lib)
    args = _attention_args()
    args.update(q_start_loc=torch.arange(3), q_seqlens=torch.ones(3, dtype=torch.int32), max_seqlen=1, window_size=8, num_sinks=2)
    args[name] = args[name].to(torch.int16)
    with pytest.raises(AssertionError, match=name):
        dl.sink_attention_fwd(**args)


def test_attention_entries():
    """Argument errors of the C entries, before any launch."""
    lib = _lib.load()

    def sink(q=16, tokens=3, batch=3, most=1, hq=4, hkv=2, d=64, dv=64, page=16, pages=4, cols=2, q_st=256, o_sh=64,
             window=8, sinks=2, scale=0.1, cap=-1.0, dtype=_lib.DTYPE_BF16):
        return lib.dlb_sink_attention(q, 16, 16, 16, 16, 16, 16, 16, batch, tokens, most, hq, hkv, d, dv, page, pages, cols,
                                      q_st, 64, 256, o_sh, 2048, 128, 64, 2048, 128, 64, 2, 0, 0, 0, 0, window, sinks, scale,
                                      cap, dtype, None, None)

    for bad in (dict(q=None), dict(q=8), dict(tokens=-1), dict(hq=3), dict(hq=258, hkv=2), dict(d=12), dict(d=136),
                dict(dv=0), dict(page=24), dict(page=8), dict(pages=0), dict(cols=0), dict(q_st=252), dict(o_sh=4),
                dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(cap=1e-30),
                dict(dtype=_lib.DTYPE_F32), dict(batch=70000), dict(cols=1 << 28), dict(most=-1)):
        assert sink(**bad) < 0 and lib.dlb_last_error().startswith(b"sink_attention"), bad
    for nothing in (dict(batch=0), dict(tokens=0), dict(most=0)):
        assert sink(**nothing) == 0

    def prefix(q=16, partial=16, batch=3, groups=2, hq=4, hkv=2, d=64, page=16, prefix_cols=2, cols=2, chunk=64, cluster=1,
               scale=0.1, cap=-1.0, dtype=_lib.DTYPE_BF16):
        return lib.dlb_shared_prefix_attention(q, 16, 16, 16, 16, 16, 16, 16, 16, partial, batch, groups, hq, hkv, d, 64,
                                               page, 4, prefix_cols, cols, 256, 64, 256, 64, 2048, 128, 64, 2048, 128, 64,
                                               2, 2, 0, 0, 0, 0, 0, chunk, cluster, scale, cap, dtype, None, None)

    for bad in (dict(q=None), dict(partial=None), dict(partial=8), dict(batch=-1), dict(groups=0), dict(groups=80000),
                dict(hq=3), dict(d=12), dict(page=8), dict(prefix_cols=0), dict(cols=0), dict(chunk=0), dict(chunk=100),
                dict(cluster=0), dict(cluster=3), dict(cluster=16),
                dict(scale=0.0), dict(cap=1e-30), dict(dtype=_lib.DTYPE_F32), dict(prefix_cols=1 << 28), dict(cols=1 << 28)):
        assert prefix(**bad) < 0 and lib.dlb_last_error().startswith(b"shared_prefix_attention"), bad
    assert prefix(batch=0) == 0
    assert lib.dlb_shared_prefix_workspace_floats(3, 4, 96, 5) == 3 * 4 * 5 * 130


def test_prefix_split_rule():
    """Chunks are whole blocks and no longer than the table; few rows are split over the SMs, many are not."""
    from dlcompiler_b200.kernels.shared_prefix_attention import _pick_prefix_split

    for tiles in (0, 1, 8, 64, 72, 296, 5000):
        for groups in (1, 3, 100):
            for blocks in (1, 2, 16, 63, 512, 1876, 30000):
                chunk, cluster = _pick_prefix_split(tiles, groups, 8, blocks)
                assert chunk % 64 == 0 and 64 <= chunk <= blocks * 64 and cluster in (1, 2, 4)
    assert _pick_prefix_split(5000, 1, 8, 512) == (512 * 64, 1)
    chunk, cluster = _pick_prefix_split(8, 1, 8, 1876)
    assert 148 < 8 * cluster * -(-1876 * 64 // chunk) <= 224


def test_tables_that_end_near_2_31_tokens():
    """Keys are counted in 32 bits, some blocks past a table's end."""
    lib = _lib.load()
    for columns in ((1 << 27) - 1, (1 << 27) - 512, 1 << 62):
        assert lib.dlb_sink_attention(16, 16, 16, 16, 16, 16, 16, 16, 3, 3, 1, 4, 2, 64, 64, 16, 4, columns, 256, 64, 256, 64, 2048,
                                      128, 64, 2048, 128, 64, 2, 0, 0, 0, 0, 8, 2, 0.1, -1.0, _lib.DTYPE_BF16, None, None) == -5
        for prefix, own in ((2, columns), (columns, 2)):
            assert lib.dlb_shared_prefix_attention(16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 3, 2, 4, 2, 64, 64, 16, 4, prefix, own, 256,
                                                   64, 256, 64, 2048, 128, 64, 2048, 128, 64, 2, 2, 0, 0, 0, 0, 0, 64, 1, 0.1, -1.0,
                                                   _lib.DTYPE_BF16, None, None) == -5


@pytest.mark.parametrize("window", [None, -1])
def test_sink_attention_has_no_code_for_no_window(no_launch, window):
    """paged_attention_fwd takes None and -1 for no window."""
    args = _attention_args()
    args.update(q_start_loc=torch.arange(3), q_seqlens=torch.ones(3, dtype=torch.int32), max_seqlen=1, num_sinks=2)
    with pytest.raises(AssertionError, match="window_size"):
        dl.sink_attention_fwd(**args, window_size=window)
