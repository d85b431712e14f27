"""Refusals of the label-distribution operators (lib/losses.py top_logits / distill_loss, lib/sampling.py, include/motifs_hip.h) that need
no device: nothing is launched."""
import ctypes
import math

import pytest
import torch

from lib import _hip
from lib.losses import TopLogits, distill_loss, top_logits
from lib.sampling import sample_labels

X = torch.zeros(4, 10)
REC = TopLogits(torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4))


def test_no_cpu_path():
    for call in (lambda: top_logits(X, 3), lambda: distill_loss(X, REC), lambda: sample_labels(X, torch.zeros(4))):
        with pytest.raises(_hip.HipKernelError, match='no CPU fallback'):
            call()


@pytest.mark.parametrize('k', [0, -1, 11, 2.0, None])
def test_top_logits_k(k):
    with pytest.raises(ValueError, match='k must be'):
        top_logits(X, k)


@pytest.mark.parametrize('T', [0.0, -1.0, math.inf, math.nan, '1', None])
def test_temperature(T):
    with pytest.raises(ValueError, match='temperature'):
        top_logits(X, 3, T)
    with pytest.raises(ValueError, match='temperature'):
        distill_loss(X, REC, T)


def test_distill_arguments():
    with pytest.raises(ValueError, match='reduction'):
        distill_loss(X, REC, reduction='batchmean')
    for scale in (math.inf, math.nan, None):
        with pytest.raises(ValueError, match='scale'):
            distill_loss(X, REC, scale=scale)
    for shape in ((4,), (4, 0), (4, 1025)):
        with pytest.raises(ValueError, match='1 to 1024 entries'):
            distill_loss(X, REC._replace(values=torch.zeros(shape)))


@pytest.mark.parametrize('kw', [dict(temperature=-0.1), dict(temperature=math.inf), dict(temperature=math.nan), dict(temperature='a'), dict(top_p=1.5), dict(top_p=-0.1),
                                dict(top_p=math.nan), dict(min_p=1.5), dict(min_p=-1.0), dict(top_k=-1), dict(top_k=2.0), dict(top_k=2 ** 31)])
def test_sample_arguments(kw):
    with pytest.raises(ValueError, match=list(kw)[0]):
        sample_labels(X, torch.zeros(4), **kw)


def test_entry_points_refuse_bad_arguments(so_path):
    """the C entry points name what is wrong and launch nothing"""
    L = ctypes.CDLL(so_path)                 # (a handle of its own: other tests put a stand-in for the library under lib._hip)
    L.mh_last_error.restype, L.mh_distill_ws_bytes.restype = ctypes.c_char_p, ctypes.c_size_t
    _hip._label_dist_argtypes(L)
    p, one, T1 = ctypes.c_void_p(4096), ctypes.c_float(1.0), ctypes.c_double(1.0)
    big = ctypes.c_longlong(10)
    bad = [L.mh_top_logits(p, 3, big, 4, 10, 3, T1, p, p, p, None), L.mh_top_logits(p, 0, big, -1, 10, 3, T1, p, p, p, None),
           L.mh_top_logits(p, 0, big, 4, 0, 1, T1, p, p, p, None), L.mh_top_logits(p, 0, big, 4, 10, 11, T1, p, p, p, None),
           L.mh_top_logits(p, 0, big, 4, 10, 0, T1, p, p, p, None), L.mh_top_logits(p, 0, big, 4, 2000, 1025, T1, p, p, p, None),
           L.mh_top_logits(p, 0, big, 4, 10, 3, ctypes.c_double(0.0), p, p, p, None), L.mh_top_logits(p, 0, big, 4, 10, 3, ctypes.c_double(math.nan), p, p, p, None),
           L.mh_top_logits(None, 0, big, 4, 10, 3, T1, p, p, p, None), L.mh_top_logits(p, 0, big, 4, 10, 3, T1, p, p, None, None)]
    z = ctypes.c_size_t(0)

    def fwd(dtype=0, rows=4, classes=10, t_dtype=0, k=3, T=1.0, logits=p, stats=p, ws=z):
        return L.mh_distill_fwd(logits, dtype, big, rows, classes, p, t_dtype, p, 0, p, k, ctypes.c_double(T), T1, None, 1, stats, p, p, p, None, p, ws, None)

    bad += [fwd(dtype=-1), fwd(rows=-1), fwd(classes=0), fwd(t_dtype=7), fwd(k=0), fwd(k=1025), fwd(T=0.0), fwd(T=math.nan), fwd(logits=None), fwd(stats=None),
            fwd(classes=1 << 20)]        # (a workspace of no bytes)

    def bwd(dtype=0, rows=4, k=3, T=1.0, grad=p, upstream=p):
        return L.mh_distill_bwd(p, dtype, big, rows, 10, p, 0, p, 0, p, k, ctypes.c_double(T), T1, None, p, p, upstream, 0, 0, grad, None)

    bad += [bwd(dtype=3), bwd(rows=-2), bwd(k=0), bwd(T=-1.0), bwd(grad=None), bwd(upstream=None)]

    def sample(dtype=0, rows=4, classes=10, logits=p, u=p, labels=p):
        return L.mh_sample_labels(logits, dtype, big, rows, classes, u, None, None, None, None, one, 0, one, one, labels, None, z, None)

    bad += [sample(dtype=9), sample(rows=-1), sample(classes=0), sample(logits=None), sample(u=None), sample(labels=None)]
    assert bad == [-1] * len(bad)
    assert b'bad argument' in L.mh_last_error()
    L.mh_sample_ws_bytes.restype = ctypes.c_size_t
    bad = [L.mh_sample_labels(p, 0, big, 4, 1 << 20, p, None, None, None, None, one, 0, one, one, p, p, z, None)]      # a workspace that is too small
    assert bad == [-1] and L.mh_sample_ws_bytes(4, 1000) == 0 and L.mh_sample_ws_bytes(4, 1 << 20) > 0
    assert L.mh_distill_ws_bytes(8, 100) == 0 and L.mh_distill_ws_bytes(8, 1 << 20) > 0
    assert L.mh_top_logits(None, 0, big, 0, 10, 3, T1, None, None, None, None) == 0 and sample(rows=0, logits=None, u=None, labels=None) == 0      # no rows: nothing to do


def test_entry_points_refuse_more_rows_than_a_launch_holds(so_path):
    L = ctypes.CDLL(so_path)
    _hip._label_dist_argtypes(L)
    p, stride = ctypes.c_void_p(4096), ctypes.c_longlong(10)
    for rows, classes in ((1 << 23, 10), (2 ** 31 - 1, 10), (1 << 22, 65537), (1 << 10, 2 ** 31 - 1)):
        assert L.mh_top_logits(p, 0, stride, rows, classes, 3, 1.0, p, p, p, None) == -1
        assert L.mh_distill_fwd(p, 0, stride, rows, classes, p, 0, p, 0, p, 3, 1.0, 1.0, None, 1, p, p, p, p, None, p, 1 << 62, None) == -1
        assert L.mh_distill_bwd(p, 0, stride, rows, classes, p, 0, p, 0, p, 3, 1.0, 1.0, None, p, p, p, 0, 0, p, None) == -1
        assert L.mh_sample_labels(p, 0, stride, rows, classes, p, None, None, None, None, 1.0, 0, 1.0, 0.0, p, None, 0, None) == -1


def test_capture_id_needs_a_place_for_its_answer(so_path):
    L = ctypes.CDLL(so_path)
    _hip._label_dist_argtypes(L)
    assert L.mh_capture_id(None, None) == -1
