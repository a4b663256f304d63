"""Generalised SDDMM front end: gsddmm and the generated u_add_v ... e_dot_v helpers
(surface of the reference's python/gs/ops/sddmm.py:35-131 and sparse.py:14-129); and, not in the
reference, rows of features moved by ids, with gradients: `embedding`, and rows sorted by expert or
node type and back, `expert_dispatch` and `expert_combine`."""
import sys
from collections import namedtuple
from itertools import product

import torch

from . import load_library
from .format import _COO

__all__ = ['gsddmm', 'embedding', 'ExpertOrder', 'expert_sort', 'expert_gather', 'expert_dispatch',
           'expert_combine']

_TARGET = {'u': 0, 'e': 1, 'v': 2, 'src': 0, 'edge': 1, 'dst': 2}


def infer_broadcast_shape(op, shp1, shp2):
    """Feature shape of the result (NumPy broadcasting; dot folds the last axis to 1)."""
    if op == "dot" and shp1[-1] != shp2[-1]:
        raise ValueError("Dot operator is only available for arrays with the same size on last "
                         "dimension, but got {} and {}.".format(shp1, shp2))
    n = max(len(shp1), len(shp2))
    p1 = (1,) * (n - len(shp1)) + tuple(shp1)
    p2 = (1,) * (n - len(shp2)) + tuple(shp2)
    for d1, d2 in zip(p1, p2):
        if d1 != d2 and d1 != 1 and d2 != 1:
            raise ValueError("Feature shapes {} and {} are not valid for broadcasting.".format(shp1, shp2))
    out = tuple(max(d1, d2) for d1, d2 in zip(p1, p2))
    return out[:-1] + (1,) if op == "dot" else out


def _pad_dims(lhs, rhs):
    """(N, 3, 1) with (E, 5, 3, 4) -> (N, 1, 3, 1): same number of feature axes."""
    if lhs.dim() != rhs.dim():
        n = max(lhs.dim(), rhs.dim())
        lhs = lhs.view((lhs.shape[0],) + (1,) * (n - lhs.dim()) + tuple(lhs.shape[1:]))
        rhs = rhs.view((rhs.shape[0],) + (1,) * (n - rhs.dim()) + tuple(rhs.shape[1:]))
    return lhs, rhs


def gsddmm(g, op, lhs_data, rhs_data, lhs_target='u', rhs_target='v', on_format=_COO):
    """x_e = op(x_lhs, x_rhs) for every edge of the Matrix `g`; returns the edge feature.

    sub is computed as add(-rhs) and div as mul(1/rhs), as the reference does
    (python/gs/ops/sparse.py:123-128)."""
    if lhs_data.device != rhs_data.device:
        raise ValueError("The operands data device don't match: {} and {}".format(
            lhs_data.device, rhs_data.device))
    if lhs_data.dtype != rhs_data.dtype:
        raise ValueError("The operands data type don't match: {} and {}".format(
            lhs_data.dtype, rhs_data.dtype))
    lhs, rhs = _pad_dims(lhs_data, rhs_data)
    if op == 'sub':
        op, rhs = 'add', -rhs
    elif op == 'div':
        op, rhs = 'mul', 1. / rhs
    squeeze = lhs.dim() == 1 and rhs.dim() == 1
    if lhs.dim() == 1:
        lhs = lhs.unsqueeze(-1)
    if rhs.dim() == 1:
        rhs = rhs.unsqueeze(-1)
    out = g._graph._CAPI_SDDMMOut(op, lhs.contiguous(), rhs.contiguous(),
                                  infer_broadcast_shape(op, lhs.shape[1:], rhs.shape[1:]),
                                  _TARGET[lhs_target], _TARGET[rhs_target], on_format)
    return out.squeeze(-1) if squeeze else out


def _make(lhs_target, rhs_target, binary_op):
    def func(g, x, y, on_format=_COO):
        return gsddmm(g, binary_op, x, y, lhs_target=lhs_target, rhs_target=rhs_target,
                      on_format=on_format)
    func.__name__ = "{}_{}_{}".format(lhs_target, binary_op, rhs_target)
    func.__doc__ = "Edge feature = {} of the {} and {} features.".format(binary_op, lhs_target, rhs_target)
    return func


for _l, _r in product("uve", "uve"):
    if _l != _r:
        for _op in ("add", "sub", "mul", "div", "dot"):
            _f = _make(_l, _r, _op)
            setattr(sys.modules[__name__], _f.__name__, _f)
            __all__.append(_f.__name__)


def embedding(weight, ids, scale=1.0, sparse_grad=False):
    """scale * weight[ids]: the rows of `weight` (2-D; float32, float16 or bfloat16) that `ids` (int32 or
    int64, any shape) name, of shape [*ids.shape, weight.shape[1]].  An id outside the table -- the -1 of
    a walker that has died, of padding -- gives a row of zeros and no gradient.

    The gradient of `weight` is summed in float32 by sorted ids, without atomics: the same bits
    every time.  With `sparse_grad` it is a coalesced sparse tensor of the rows that were met (for
    torch.optim.SparseAdam and SGD); the backward pass then waits for how many there are, and
    cannot be recorded into a graph.

        input_nodes, blocks = gs.sample_layers(A, seeds, [15, 10, 5])
        h = gs.ops.embedding(node_table, input_nodes, sparse_grad=True)
    """
    load_library()
    return torch.ops.gs_ops._CAPI_Embedding(weight, ids, scale, sparse_grad)


# order: int32 [items], the item (token * choices + choice) at each place, -1 behind the last;
# place: int32 like the experts, where each item lies, -1 where it names no expert;
# offsets: int64 [experts + 1], where each expert's rows begin and the last one's end
ExpertOrder = namedtuple('ExpertOrder', ['order', 'place', 'offsets'])


def expert_sort(experts, num_experts):
    """The items of `experts` ([tokens] or [tokens, choices], int32 or int64) sorted by expert, stably:
    an ExpertOrder.  An item whose expert lies outside [0, num_experts) -- a choice that found no
    room -- has no place.  With one choice each, experts may as well be node types or relations."""
    load_library()
    return ExpertOrder(*torch.ops.gs_ops._CAPI_ExpertSort(experts, num_experts))


def expert_gather(x, order):
    """A copy of row t of `x` ([tokens, dim]) at every place of token t: [items, dim], the rows of expert e
    from offsets[e] to offsets[e + 1], zeros behind the last.  Differentiable."""
    load_library()
    return torch.ops.gs_ops._CAPI_ExpertGather(x, order.order, order.place, order.offsets)


def expert_dispatch(x, experts, num_experts):
    """expert_sort and expert_gather in one call: (rows, ExpertOrder)."""
    load_library()
    rows, order, place, offsets = torch.ops.gs_ops._CAPI_ExpertDispatch(x, experts, num_experts)
    return rows, ExpertOrder(order, place, offsets)


def expert_combine(y, order, weights=None):
    """Row t: the sum over token t's choices k of weights[t, k] * y[place[t, k]] (`weights`: like
    order.place, float32 or of y's type; None: ones), in float32, rounded once; a choice without a
    place adds nothing.  Differentiable in `y` and `weights`.

        rows, order = gs.ops.expert_dispatch(x, experts, num_experts)
        y, at = torch.zeros_like(rows), order.offsets.tolist()
        for e, net in enumerate(nets):
            y[at[e]:at[e + 1]] = net(rows[at[e]:at[e + 1]])
        out = gs.ops.expert_combine(y, order, weights)
    """
    load_library()
    return torch.ops.gs_ops._CAPI_ExpertCombine(y, order.order, order.place, order.offsets, weights)
