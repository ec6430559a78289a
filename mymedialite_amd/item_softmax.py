"""The softmax over the catalogue of a matrix-factorization model, on torch tensors in HBM.

``item_log_probs`` gives the log probability of given items, the log normaliser, the entropy and the
likeliest items of a batch of users; ``item_log_probs_grad`` the gradient of a loss on them.  Both
run the HIP kernels of libmml_hip.so on torch's current stream of the factors' device and return
without waiting; there is no CPU path, and results carry no autograd graph.  (BPRMF.log_probs and
WRMF.log_probs are the same for a trained recommender, on host arrays.)
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N
from ._native import ItemLogProbs

_DTYPES = {torch.float32: N.DTYPE_F32, torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_F16}


def _stream(index):
    """torch's current stream of device `index` as a pointer"""
    return torch._C._cuda_getCurrentRawStream(index)


def _factors(x, name):
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError(f"{name} must be a 2-D tensor")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    # a row stride under a row's length (an expanded tensor) is laid out
    row, step = x.stride()
    return x if step == 1 and row >= x.shape[1] else x.contiguous()


def _vector(x, name, dtype, n, index):
    """x and its address"""
    if x is None:
        return None, None
    if not isinstance(x, torch.Tensor) or x.dim() != 1 or x.dtype != dtype:
        raise ValueError(f"{name} must be a 1-D {dtype} tensor")
    if n is not None and x.shape[0] != n:
        raise ValueError(f"{name} has {x.shape[0]} entries, expected {n}")
    if x.get_device() != index:
        raise ValueError(f"{name} is on {x.device}, the factors are on cuda:{index}")
    if x.stride(0) != 1 and x.shape[0] > 1:
        x = x.contiguous()
    return x, x.data_ptr()


def _arguments(user_factors, item_factors, item_bias, items, users, exclude, n_top):
    """(mml_item_softmax_args, the device's index, the tensors that the arguments point to)"""
    U, V = _factors(user_factors, "user_factors"), _factors(item_factors, "item_factors")
    if U.dtype != V.dtype:
        raise ValueError("user_factors and item_factors must have one dtype")
    index = U.get_device()
    if index != V.get_device():
        raise ValueError("user_factors and item_factors must be on one device")
    (n_users, k), (n_items, kv) = U.shape, V.shape
    if k != kv:
        raise ValueError(f"{k} user factors, {kv} item factors")
    bias, bias_at = _vector(item_bias, "item_bias", torch.float32, n_items, index)
    users, users_at = _vector(users, "users", torch.int32, None, index)
    rows = n_users if users is None else users.shape[0]
    items, items_at = _vector(items, "items", torch.int32, rows, index)
    off = ex = off_at = ex_at = None
    if exclude is not None:
        off, off_at = _vector(exclude[0], "exclude[0]", torch.int64, n_users + 1, index)
        ex, ex_at = _vector(exclude[1], "exclude[1]", torch.int32, None, index)
    a = N.ItemSoftmaxArgs(
        _DTYPES[U.dtype], k, rows, n_users, n_items, U.data_ptr(), V.data_ptr(),
        max(U.stride(0), k), max(V.stride(0), k), bias_at, users_at, items_at, off_at, ex_at,
        0 if ex is None else ex.shape[0], int(n_top))
    return a, index, (U, V, bias, users, items, off, ex)


def _workspace(a, grad, device):
    n = ctypes.c_int64(0)
    N.check(N.lib().mml_item_log_probs_workspace(ctypes.byref(a), grad, ctypes.byref(n)))
    return torch.empty(max(n.value, 256), dtype=torch.uint8, device=device)


def item_log_probs(user_factors, item_factors, item_bias=None, items=None, users=None,
                   exclude=None, n_top=0) -> ItemLogProbs:
    """The softmax over the items' scores <U_u, V_j> + b_j for every row (mml_item_log_probs_device).

    user_factors [n_users, k], item_factors [n_items, k]: float32, bfloat16 or float16, k <= 256;
    item_bias [n_items] float32; users [rows] int32: the rows' users (default: all, in order);
    items [rows] int32: the given items, -1 for none; exclude: (offsets [n_users + 1] int64, items
    int32), the CSR of every user's excluded items (Feedback.user_matrix); n_top <= 128."""
    a, index, keep = _arguments(user_factors, item_factors, item_bias, items, users, exclude, n_top)
    dev, rows, n_top = keep[0].device, a.n_rows, a.n_top
    ws = _workspace(a, 0, dev)
    log_probs, log_norm, entropy = torch.empty((3, rows), dtype=torch.float32, device=dev).unbind()
    p = log_probs.data_ptr()
    ids = lp = ids_at = lp_at = None
    if n_top:
        ids = torch.empty((rows, n_top), dtype=torch.int32, device=dev)
        lp = torch.empty((rows, n_top), dtype=torch.float32, device=dev)
        ids_at, lp_at = ids.data_ptr(), lp.data_ptr()
    N.check(N.lib().mml_item_log_probs_device(
        ctypes.byref(a), p, p + 4 * rows, p + 8 * rows, ids_at, lp_at, ws.data_ptr(), ws.shape[0],
        index, _stream(index)))
    return ItemLogProbs(log_probs, log_norm, entropy, ids, lp)


def item_log_probs_grad(user_factors, item_factors, item_bias=None, items=None, *, log_norm,
                        entropy=None, grad_log_probs=None, grad_entropy=None, users=None,
                        exclude=None):
    """(dL/dU [rows, k], dL/dV [n_items, k], dL/db [n_items]) of a loss with the given derivatives
    by item_log_probs' log_probs and entropy (mml_item_log_probs_grad_device).  The first seven
    arguments are those of that call, log_norm and entropy its results.  dL/dU has one row per row
    of the batch; the factors' gradients have the factors' type, dL/db is float32."""
    a, index, keep = _arguments(user_factors, item_factors, item_bias, items, users, exclude, 0)
    U, V = keep[0], keep[1]
    dev, rows, k = U.device, a.n_rows, a.num_factors
    if log_norm is None:
        raise ValueError("log_norm is required")
    f32 = torch.float32
    log_norm, norm_at = _vector(log_norm, "log_norm", f32, rows, index)
    entropy, entropy_at = _vector(entropy, "entropy", f32, rows, index)
    grad_log_probs, glp_at = _vector(grad_log_probs, "grad_log_probs", f32, rows, index)
    grad_entropy, gent_at = _vector(grad_entropy, "grad_entropy", f32, rows, index)
    ws = _workspace(a, 1, dev)
    gu = torch.empty((rows, k), dtype=U.dtype, device=dev)
    gv = torch.empty((a.n_items, k), dtype=U.dtype, device=dev)
    gb = torch.empty(a.n_items, dtype=f32, device=dev)
    N.check(N.lib().mml_item_log_probs_grad_device(
        ctypes.byref(a), norm_at, entropy_at, glp_at, gent_at, gu.data_ptr(), k, gv.data_ptr(), k,
        gb.data_ptr(), ws.data_ptr(), ws.shape[0], index, _stream(index)))
    return gu, gv, gb
