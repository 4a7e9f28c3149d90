"""The vocabulary head's host side: struct layout, sizes and refusals, without a GPU."""
import ctypes
import os
import subprocess

import pytest
import torch

import gpusparse._lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def view(T=100, V=500, D=64, dtype=L.W_BF16, ldh=None, ldw=None, ptr=4096):
    v = L.VocabView()
    v.T, v.V, v.D, v.dtype = T, V, D, dtype
    v.ld_hidden, v.ld_weight = ldh if ldh is not None else D, ldw if ldw is not None else D
    v.hidden = v.weight = ptr
    return v


def test_view_layout_matches_the_header(tmp_path):
    names = [n for n, _ in L.VocabView._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "gpusparse.h"\nint main(void) {\n'
                   '  printf("size %zu\\n", sizeof(gsp_vocab_view));\n'
                   + "".join(f'  printf("{n} %zu\\n", offsetof(gsp_vocab_view, {n}));\n' for n in names)
                   + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    got = dict(line.split() for line in subprocess.check_output([str(exe)], text=True).splitlines())
    assert int(got["size"]) == ctypes.sizeof(L.VocabView)
    for n in names:
        assert int(got[n]) == getattr(L.VocabView, n).offset


def test_sizes():
    lib = L.lib()
    for T in (0, 1, 255, 256, 257, 16384):
        v = view(T=T, V=30522, D=768)
        for kind in (L.VOCAB_CE, L.VOCAB_DISTILL, L.VOCAB_HEAD):
            assert lib.gsp_vocab_state_bytes(ctypes.byref(v), 10, kind) > T * 768 * 2
            assert lib.gsp_vocab_ws_bytes(ctypes.byref(v), 10, kind, 0) > 0
            back = lib.gsp_vocab_ws_bytes(ctypes.byref(v), 10, kind, 1)
            assert 0 < back < (700 << 20)         # a piece of at most 512 MiB, and dH in fp32
    # rows a tensor map cannot describe are copied: the state holds the copy
    a = lib.gsp_vocab_state_bytes(ctypes.byref(view()), 0, L.VOCAB_CE)
    for odd in (view(ldw=65), view(ptr=4098), view(D=63)):
        assert lib.gsp_vocab_state_bytes(ctypes.byref(odd), 0, L.VOCAB_CE) >= a + 500 * 64 * 2


@pytest.mark.parametrize("bad", [
    dict(dtype=L.W_F32), dict(dtype=L.W_U8), dict(T=-1), dict(V=0), dict(D=0), dict(ldh=63), dict(ldw=1),
    dict(T=(1 << 30) + 1),
])
def test_bad_views_are_refused(bad):
    lib = L.lib()
    v = view(**bad)
    assert lib.gsp_vocab_ws_bytes(ctypes.byref(v), 0, L.VOCAB_CE, 0) == -L.GSP_ERR_ARG
    assert lib.gsp_vocab_state_bytes(ctypes.byref(v), 0, L.VOCAB_CE) == -L.GSP_ERR_ARG
    fake = ctypes.c_void_p(4096)
    rc = lib.gsp_vocab_ce(ctypes.byref(v), fake, -100, 2, fake, fake, 1 << 40, fake, 1 << 40, None)
    assert rc == L.GSP_ERR_ARG and lib.gsp_last_error()


def test_bad_calls_are_refused_before_any_launch():
    lib = L.lib()
    v, fake, big = view(), ctypes.c_void_p(4096), 1 << 40
    ref = ctypes.byref(v)
    sb = lib.gsp_vocab_state_bytes(ref, 0, L.VOCAB_CE)
    wb = lib.gsp_vocab_ws_bytes(ref, 0, L.VOCAB_CE, 0)
    bb = lib.gsp_vocab_ws_bytes(ref, 0, L.VOCAB_CE, 1)
    E = L.GSP_ERR_ARG
    assert lib.gsp_vocab_ce(ref, fake, -100, 3, fake, fake, big, fake, big, None) == E
    assert lib.gsp_vocab_ce(ref, fake, -100, 2, None, fake, big, fake, big, None) == E
    assert lib.gsp_vocab_ce(ref, None, -100, 2, fake, fake, big, fake, big, None) == E
    assert lib.gsp_vocab_ce(ref, fake, -100, 2, fake, fake, sb - 1, fake, wb, None) == E
    assert lib.gsp_vocab_ce(ref, fake, -100, 2, fake, fake, sb, fake, wb - 1, None) == E
    assert lib.gsp_vocab_ce(ref, fake, -100, 2, fake, None, sb, fake, wb, None) == E
    for K, tau in ((0, 1.0), (1025, 1.0), (4, 0.0), (4, float("inf")), (4, float("nan"))):
        assert lib.gsp_vocab_distill(ref, fake, fake, K, tau, 2, fake, fake, big, fake, big, None) == E
        assert lib.gsp_vocab_loss_backward(ref, L.VOCAB_DISTILL, K, tau, 2, fake, fake, fake, fake, fake, big, fake,
                                           big, None) == E
    assert lib.gsp_vocab_loss_backward(ref, L.VOCAB_HEAD, 0, 1.0, 2, fake, fake, fake, fake, fake, big, fake, big, None) == E
    assert lib.gsp_vocab_loss_backward(ref, L.VOCAB_CE, 0, 1.0, 2, fake, fake, fake, fake, fake, sb, fake, bb - 1, None) == E
    assert lib.gsp_vocab_loss_backward(ref, L.VOCAB_CE, 0, 1.0, 2, None, fake, fake, fake, fake, sb, fake, bb, None) == E
    odd = ctypes.c_void_p(4096 + 16)                    # gradients that are not 32-byte aligned
    assert lib.gsp_vocab_loss_backward(ref, L.VOCAB_CE, 0, 1.0, 2, fake, odd, fake, fake, fake, sb, fake, bb, None) == E
    assert lib.gsp_sparse_head_backward(ref, 10, fake, fake, fake, fake, odd, fake, fake, big, fake, big, None) == E
    assert lib.gsp_sparse_head(ref, 0, None, fake, None, fake, big, fake, big, None) == E
    assert lib.gsp_sparse_head(ref, 33, None, fake, None, fake, big, fake, big, None) == E      # 100 tokens
    assert lib.gsp_sparse_head(ref, 10, None, None, None, fake, big, fake, big, None) == E
    many = view(T=70000)
    assert lib.gsp_sparse_head(ctypes.byref(many), 1, None, fake, None, fake, big, fake, big, None) == E
    assert lib.gsp_sparse_head_backward(ref, 10, fake, None, fake, fake, fake, fake, fake, big, fake, big, None) == E
    assert lib.gsp_dense_rows_count(None, 3, 5, 0.0, fake, None) == E
    assert lib.gsp_dense_rows_fill(fake, 3, 0, 0.0, fake, fake, fake, None) == E


@pytest.mark.parametrize("off", [2, 16, 128])
def test_unaligned_buffers_are_refused(off):
    lib = L.lib()
    ref, fake, odd, big = ctypes.byref(view()), ctypes.c_void_p(4096), ctypes.c_void_p(4096 + off), 1 << 40
    for st, ws in ((odd, fake), (fake, odd)):
        for rc in (lib.gsp_vocab_ce(ref, fake, -100, 2, fake, st, big, ws, big, None),
                   lib.gsp_vocab_distill(ref, fake, fake, 4, 1.0, 2, fake, st, big, ws, big, None),
                   lib.gsp_vocab_loss_backward(ref, L.VOCAB_CE, 0, 1.0, 2, fake, fake, fake, fake, st, big, ws, big, None),
                   lib.gsp_sparse_head(ref, 10, None, fake, None, st, big, ws, big, None),
                   lib.gsp_sparse_head_backward(ref, 10, fake, fake, fake, fake, fake, fake, st, big, ws, big, None)):
            assert rc == L.GSP_ERR_ARG and b"256" in lib.gsp_last_error()


def test_host_tensors_are_refused():
    import gpusparse
    h, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        gpusparse.vocab_cross_entropy(h, w, t)
    with pytest.raises(RuntimeError):
        gpusparse.topk_distillation(h, w, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        gpusparse.sparse_head(h[None], w)


def test_tangents_are_noticed():
    """A dual tensor needs no gradient; its call still belongs in the autograd function, which
    refuses it, and not in one that drops the tangent."""
    import torch.autograd.forward_ad as fwd
    from gpusparse import head
    x, w, b = torch.ones(2, 3), torch.ones(4, 3), torch.ones(4)
    assert not head._differentiated(x, w, b) and head._differentiated(x, w, torch.ones(4, requires_grad=True))
    with fwd.dual_level():
        assert not head._differentiated(x, w, None)
        with torch.no_grad():
            assert head._differentiated(fwd.make_dual(x, x), w, None)
            assert head._differentiated(x, w, fwd.make_dual(b, b))
            assert not head._differentiated(x, w, torch.ones(4, requires_grad=True))


def test_temperatures_that_leave_fp32_are_refused():
    """The square or the reciprocal would be 0, infinite or short of bits, and the losses NaN."""
    lib = L.lib()
    ref, fake, big = ctypes.byref(view()), ctypes.c_void_p(4096), 1 << 40
    for tau in (1e-45, 1e-39, 1e-30, 1.08e-19, 1.9e19, 1e30, -1.0, -1e-30):
        assert lib.gsp_vocab_distill(ref, fake, fake, 4, tau, 2, fake, fake, big, fake, big, None) == L.GSP_ERR_ARG
        assert b"temperature" in lib.gsp_last_error()
        assert lib.gsp_vocab_loss_backward(ref, L.VOCAB_DISTILL, 4, tau, 2, fake, fake, fake, fake, fake, big, fake, big,
                                           None) == L.GSP_ERR_ARG
        assert b"temperature" in lib.gsp_last_error()
    for tau in (1.1e-19, 1.8e19):         # accepted: the next check, of the buffers, is the one that refuses
        assert lib.gsp_vocab_distill(ref, fake, fake, 4, tau, 2, fake, fake, 0, fake, big, None) == L.GSP_ERR_ARG
        assert b"state" in lib.gsp_last_error()
