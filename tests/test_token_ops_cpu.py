"""Refusals of the token operators that need no GPU: argument checks of the Python entry points and of the C entries, which look at
everything they can on the host before a device is touched."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def N():
    from multi_modal_amd import _native
    _native.load_library()
    return _native


@pytest.mark.parametrize("kw", [dict(sections=[]), dict(sections=[1] * 5), dict(sections=[0, 0]), dict(sections=[-1, 4]), dict(sections=[513]),
                                dict(sections=[4], ladder="both"), dict(sections=[4], pairing="third"), dict(sections=[4], base=0.0),
                                dict(sections=[4], base=math.inf), dict(sections=[4], base=math.nan)])
def test_rotary_constructor_refuses(N, kw):
    from multi_modal_amd.rotary import Rotary
    with pytest.raises(ValueError):
        Rotary(**kw)


def test_grid_positions():
    from multi_modal_amd.rotary import grid_positions
    p = grid_positions(2, 3)
    assert p.dtype == torch.int32 and p.tolist() == [[0, 0, 0, 1, 1, 1], [0, 1, 2, 0, 1, 2]]
    assert grid_positions(4, 0, 2).shape == (3, 0)
    with pytest.raises(ValueError):
        grid_positions()


def test_rotary_entries_refuse(N):
    lib = N.load_library()
    h = ctypes.c_void_p()
    def create(sections, ladder=0, pairing=0, base=10000.0):
        s = (ctypes.c_int32 * max(1, len(sections)))(*sections)
        return lib.mmfe_rotary_create(len(sections), s, ladder, pairing, base, 0, ctypes.byref(h))
    for args in (([],), ([1] * 5,), ([0],), ([-3, 5],), ([300, 300],), ([4], 2), ([4], 0, 2), ([4], 0, 0, -1.0), ([4], 0, 0, math.nan)):
        assert create(*args) == -1 and h.value is None, args
    assert lib.mmfe_rotary_create(1, None, 0, 0, 10000.0, 0, ctypes.byref(h)) == -1
    assert lib.mmfe_rotary_run(None, None, None) == -1
    assert lib.mmfe_rotary_destroy(None) == 0
    if not torch.cuda.is_available():
        assert create([4]) == -2                       # no device: no CPU path


def test_struct_sizes_match_header(N):
    """The ctypes structures have the C layout (8-byte members on 8-byte boundaries, no padding inside)."""
    assert ctypes.sizeof(N.RotaryArgs) == 8 * 4 + 2 * 8 + 4 * 8 + 12 * 8 + 8 + 3 * 8


def clip(N, ptrs, numels, dtypes, outs=None, out_dtypes=None, kind=2, max_norm=1.0, partials=64, norm=64):
    lib, n = N.load_library(), len(ptrs)
    vp, i64, i32 = ctypes.c_void_p * max(1, n), ctypes.c_int64 * max(1, n), ctypes.c_int32 * max(1, n)
    return lib.mmfe_grad_clip(n, vp(*ptrs), i64(*numels), i32(*dtypes), None if outs is None else vp(*outs),
                              None if out_dtypes is None else i32(*out_dtypes), kind, max_norm, partials, norm, 99, None)


def test_clip_entry_refuses(N):
    """Every call names device 99: one that passes the checks is refused for that (-2 or -3), nothing is launched."""
    A, B = 1 << 20, 1 << 21
    ok = clip(N, [A, B], [100, 50], [0, 0], [A, B], [0, 0])
    assert ok not in (0, -1)
    assert clip(N, [A, B], [100, 50], [0, 2], [A, B], [0, 2], kind=0) == ok
    assert clip(N, [A, A + 200], [100, 50], [2, 0], [A, A + 200], [2, 0]) == ok          # behind one another
    bad = [
        clip(N, [A, B], [100, 50], [0, 0], [A, B], [0, 0], kind=1),
        clip(N, [A, B], [100, -1], [0, 0], [A, B], [0, 0]),
        clip(N, [A, B], [100, 50], [0, 3], [A, B], [0, 3]),
        clip(N, [A, None], [100, 50], [0, 0]),
        clip(N, [A, B + 2], [100, 50], [0, 0]),                                           # float32 off its alignment
        clip(N, [A, B], [100, 50], [0, 0], [A, B], [0, 0], max_norm=-1.0),
        clip(N, [A, B], [100, 50], [0, 0], [A, B], [0, 0], max_norm=math.nan),
        clip(N, [A, B], [100, 50], [0, 0], [A, None], [0, 0]),
        clip(N, [A, B], [100, 50], [0, 0], [A, B], None),
        clip(N, [A, A], [100, 100], [0, 0], [A, A], [0, 0]),                              # the same gradient twice
        clip(N, [A, A + 396], [100, 50], [0, 0], [A, A + 396], [0, 0]),                   # one element shared
        clip(N, [A], [100], [0], [A + 4], [0]),                                           # result shifted over its input
        clip(N, [A], [100], [0], [A], [1]),                                               # in place with another type
        clip(N, [A, B], [100, 50], [0, 0], partials=None),
        clip(N, [A, B], [100, 50], [0, 0], norm=None),
    ]
    assert bad == [-1] * len(bad)
    assert clip(N, [A, A], [100, 100], [0, 0]) == ok                                      # a norm alone may read a tensor twice
    assert N.load_library().mmfe_grad_partials(-1) == 0


def test_wrappers_refuse(N):
    from multi_modal_amd.gradients import clip_grad_norm, grad_norm
    x = torch.ones(4)
    with pytest.raises(ValueError, match="norm_type"):
        clip_grad_norm([x], 1.0, norm_type=1.0)
    with pytest.raises(ValueError, match="norm_type"):
        grad_norm([x], norm_type=3)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm([x], bad)
    if not torch.cuda.is_available():
        with pytest.raises(N.MmfeError):
            clip_grad_norm([x], 1.0)


def test_share_of_views():
    """What inplace=True asks about its two tensors: cuts of one packed projection share nothing, overlapping cuts do."""
    from multi_modal_amd.rotary import _share
    qkv = torch.zeros(2, 5, 12, 8)
    assert not _share(qkv[:, :, :4], qkv[:, :, 4:8])
    assert _share(qkv[:, :, :5], qkv[:, :, 4:8])
    assert _share(qkv[:, :, :4], qkv[:, :, :4])
    assert not _share(torch.zeros(1, 2, 3, 4), torch.zeros(1, 2, 3, 4))
    assert _share(qkv[:, 1:, :4], qkv[:, :-1, :4])
    flat = torch.zeros(200)
    a = flat.as_strided((1, 5, 2, 8), (0, 16, 8, 1))
    b = flat.as_strided((1, 5, 2, 8), (0, 16, 8, 1), 16)      # the same tokens, one further on
    assert _share(a, b)


def test_clip_entry_takes_empty_tensors(N):
    """Tensors without elements have no address: two of them share nothing, whatever their types."""
    assert clip(N, [None, 1 << 20, None], [0, 10, 0], [0, 0, 1], [None, 1 << 20, None], [1, 0, 1]) not in (0, -1)
