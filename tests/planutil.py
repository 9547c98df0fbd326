"""The host-side plans of the prompt operators, asked of the built library:
which kernel, tile and splits a call of the given sizes takes. Tests use them
to state which path a shape runs, so that a change of the plans' cost figures
cannot take a path out of the tests unseen."""
import ctypes
from collections import namedtuple

_I = ctypes.c_int


class _Linear(ctypes.Structure):
    _fields_ = [(n, _I) for n in ("tm", "tn", "small", "splits", "split_stages")]


class _Attn(ctypes.Structure):
    _fields_ = [(n, _I) for n in ("many", "groups", "splits", "tail", "tail_tiles")] + [("part_rows", ctypes.c_int64)]


LinearPlan = namedtuple("LinearPlan", "tm tn small split")
AttnPlan = namedtuple("AttnPlan", "many groups splits tail tail_tiles")


def linear_plan(qimg, x_dtype, M, N, K, gated):
    """tm = 0: the kernels of few rows; split: the sum over K goes over workgroups."""
    f = qimg.lib()["_ZN4qimg17linear_fused_planEiiiib"]
    f.restype, f.argtypes = _Linear, [_I, _I, _I, _I, ctypes.c_bool]
    p = f(x_dtype, M, K, N, bool(gated))
    return LinearPlan(p.tm, p.tn, bool(p.small), p.splits > 1)


def attn_plan(qimg, total_q, total_k, batch, hq, hk, d, causal):
    """many: tiles of 128 rows (with `groups` wave groups), else of 32; splits: most key ranges."""
    f = qimg.lib()["_ZN4qimg16attn_varlen_planEiiiiiib"]
    f.restype, f.argtypes = _Attn, [_I] * 6 + [ctypes.c_bool]
    p = f(total_q, total_k, batch, hq, hk, d, bool(causal))
    return AttnPlan(bool(p.many), p.groups, p.splits, p.tail, p.tail_tiles)
