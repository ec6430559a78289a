"""The softmax over the catalogue of a matrix-factorization model, on torch tensors in HBM.

``item_log_probs`` gives the log probability of given items, the log normaliser, the entropy and the
likeliest items of a batch of users; ``item_log_probs_grad`` the gradient of a loss on them.  Both
run the HIP kernels of libmml_hip.so on torch's current stream of the factors' device and return
without waiting; there is no CPU path.  (BPRMF.log_probs and WRMF.log_probs are the same for a
trained recommender, on host arrays.)
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N
from ._native import ItemLogProbs

_DTYPES = {torch.float32: N.DTYPE_F32, torch.bfloat16: N.DTYPE_BF16, torch.float16: N.DTYPE_F16}


def _factors(x, name):
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError(f"{name} must be a 2-D tensor")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    # a row stride under a row's length (an expanded tensor) is laid out
    return x if x.stride(1) == 1 and x.stride(0) >= x.shape[1] else x.contiguous()


def _vector(x, name, dtype, n, device):
    if x is None:
        return None
    if not isinstance(x, torch.Tensor) or x.dim() != 1 or x.dtype != dtype:
        raise ValueError(f"{name} must be a 1-D {dtype} tensor")
    if n is not None and x.shape[0] != n:
        raise ValueError(f"{name} has {x.shape[0]} entries, expected {n}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, the factors are on {device}")
    return x if x.stride(0) == 1 or x.numel() < 2 else x.contiguous()


def _ptr(x):
    return None if x is None else x.data_ptr()


def _arguments(user_factors, item_factors, item_bias, items, users, exclude, n_top):
    """(mml_item_softmax_args, the tensors that it points to)"""
    U, V = _factors(user_factors, "user_factors"), _factors(item_factors, "item_factors")
    if U.dtype != V.dtype:
        raise ValueError("user_factors and item_factors must have one dtype")
    if U.device != V.device:
        raise ValueError("user_factors and item_factors must be on one device")
    if U.shape[1] != V.shape[1]:
        raise ValueError(f"{U.shape[1]} user factors, {V.shape[1]} item factors")
    dev = U.device
    bias = _vector(item_bias, "item_bias", torch.float32, V.shape[0], dev)
    users = _vector(users, "users", torch.int32, None, dev)
    rows = U.shape[0] if users is None else users.shape[0]
    items = _vector(items, "items", torch.int32, rows, dev)
    off = ex = None
    if exclude is not None:
        off = _vector(exclude[0], "exclude[0]", torch.int64, U.shape[0] + 1, dev)
        ex = _vector(exclude[1], "exclude[1]", torch.int32, None, dev)
    n_top = int(n_top)
    a = N.ItemSoftmaxArgs(
        _DTYPES[U.dtype], U.shape[1], rows, U.shape[0], V.shape[0], U.data_ptr(), V.data_ptr(),
        max(U.stride(0), U.shape[1]), max(V.stride(0), V.shape[1]), _ptr(bias), _ptr(users),
        _ptr(items), _ptr(off), _ptr(ex), 0 if ex is None else ex.shape[0], n_top)
    return a, (U, V, bias, users, items, off, ex)


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
    a, keep = _arguments(user_factors, item_factors, item_bias, items, users, exclude, n_top)
    dev, rows, n_top = keep[0].device, a.n_rows, a.n_top
    ws = _workspace(a, 0, dev)
    out = torch.empty((3, rows), dtype=torch.float32, device=dev)
    ids = lp = None
    if n_top:
        ids = torch.empty((rows, n_top), dtype=torch.int32, device=dev)
        lp = torch.empty((rows, n_top), dtype=torch.float32, device=dev)
    p = out.data_ptr()
    N.check(N.lib().mml_item_log_probs_device(
        ctypes.byref(a), p, p + 4 * rows, p + 8 * rows, _ptr(ids), _ptr(lp), ws.data_ptr(),
        ws.numel(), dev.index, torch.cuda.current_stream(dev).cuda_stream))
    return ItemLogProbs(out[0], out[1], out[2], ids, lp)


def item_log_probs_grad(user_factors, item_factors, item_bias=None, items=None, *, log_norm,
                        entropy=None, grad_log_probs=None, grad_entropy=None, users=None,
                        exclude=None):
    """(dL/dU [rows, k], dL/dV [n_items, k], dL/db [n_items]) of a loss with the given derivatives
    by item_log_probs' log_probs and entropy (mml_item_log_probs_grad_device).  The first seven
    arguments are those of that call, log_norm and entropy its results.  dL/dU has one row per row
    of the batch; the factors' gradients have the factors' type, dL/db is float32."""
    a, keep = _arguments(user_factors, item_factors, item_bias, items, users, exclude, 0)
    U, V = keep[0], keep[1]
    dev, rows = U.device, a.n_rows
    vec = [_vector(x, n, torch.float32, rows, dev) for x, n in (
        (log_norm, "log_norm"), (entropy, "entropy"), (grad_log_probs, "grad_log_probs"),
        (grad_entropy, "grad_entropy"))]
    if vec[0] is None:
        raise ValueError("log_norm is required")
    ws = _workspace(a, 1, dev)
    k = a.num_factors
    gu = torch.empty((rows, k), dtype=U.dtype, device=dev)
    gv = torch.empty((V.shape[0], k), dtype=U.dtype, device=dev)
    gb = torch.empty(V.shape[0], dtype=torch.float32, device=dev)
    N.check(N.lib().mml_item_log_probs_grad_device(
        ctypes.byref(a), *(_ptr(x) for x in vec), gu.data_ptr(), k, gv.data_ptr(), k,
        gb.data_ptr(), ws.data_ptr(), ws.numel(), dev.index,
        torch.cuda.current_stream(dev).cuda_stream))
    return gu, gv, gb
