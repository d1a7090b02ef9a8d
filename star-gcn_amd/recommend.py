"""Answers out of the whole item catalogue: scores of a user's row against every item's row in 8 bits, and items drawn from
them.  The reference scores given (user, item) pairs only (experiments/STAR-GCN.py:428-438).

    net.eval()
    plan = net.make_plan(graph, full_node_ids=graph.node_ids_dict)            # every node: the whole catalogue
    with torch.no_grad():
        users, items = net.rating_rows(plan)
    user_ids, item_ids = net.rating_ids(plan)                                 # the nodes that the rows belong to
    head = CatalogueHead(items, item_ids=item_ids)                            # once per refresh of the item rows
    ids, prob = head.draw(users[rows], torch.rand(len(rows), device=users.device), temperature=0.7, top_k=100, seen=seen)
    # ids: items of the graph; row i of the answer is user user_ids[rows[i]]
"""
import torch

from . import _lib as L
from . import ops


def _mask_pairs(scores, rows, items):
    """scores[rows[i], items[i]] = -inf; pairs outside the scores are passed over.  A minimum with +inf changes nothing, so this
    needs neither a look at the indices on the host nor a list of the valid ones, and can be captured."""
    if rows.is_floating_point() or items.is_floating_point() or torch.bool in (rows.dtype, items.dtype):
        raise L.StarGCNError("CatalogueHead: seen is a pair of index tensors, got %s and %s" % (rows.dtype, items.dtype))
    try:
        rows, items = torch.broadcast_tensors(rows, items)
    except RuntimeError:
        raise L.StarGCNError("CatalogueHead: seen's shapes %s and %s do not go together" % (tuple(rows.shape), tuple(items.shape)))
    if not scores.numel() or not rows.numel():
        return
    m, n = scores.shape
    rows, items = rows.reshape(-1).long(), items.reshape(-1).long()
    inside = (rows >= 0) & (rows < m) & (items >= 0) & (items < n)
    value = torch.full(inside.shape, float("inf"), dtype=scores.dtype, device=scores.device).masked_fill_(inside, -float("inf"))
    scores.view(-1).scatter_reduce_(0, torch.where(inside, rows * n + items, torch.zeros_like(rows)), value, "amin")


class CatalogueHead(object):
    """The item rows as 8-bit codes with one scale an item (a quarter of the fp32 rows' bytes).  A score is the inner product of
    the dequantised rows, summed exactly: |score - <user, item>| <= sum of |u_k| s_i / 2 + |i_k| s_u / 2 + s_u s_i / 4 over k, s = max|row| / 127.

    item_ids (items): the ids of the rows, whole numbers that are all different, e.g. the second of Net.rating_ids; draw
    then answers with them, in their type, and takes them in `seen`.  Without, an item's id is its row.  Scores keep the rows' order.

    bias (items) fp32 is added to every score.  With norm_weight (width), user rows pass through the root-mean-square norm
    first, optionally with a residual: the scores' scale, and so what `temperature` means, is then the same for every user."""

    def __init__(self, item_rows, bias=None, norm_weight=None, eps=1e-6, item_ids=None):
        self.codes, self.scale = ops.quantize_rows(item_rows.detach())
        self.bias, self.norm_weight, self.eps = bias, norm_weight, eps
        self.items = self.codes.shape[0]
        self.item_ids = None if item_ids is None else item_ids.clone()
        if item_ids is not None:
            L.require_current_gpu(item_ids)
            if item_ids.dtype not in (torch.int32, torch.int64) or item_ids.shape != (self.items,):
                raise L.StarGCNError("CatalogueHead: item_ids of shape (%d,) and type int32 or int64 expected, got %s of %s" %
                                     (self.items, tuple(item_ids.shape), item_ids.dtype))
            self._sorted_ids, self._sorted_rows = item_ids.long().sort()
            if self.items and (int(self._sorted_ids[0]) < 0 or bool((self._sorted_ids[1:] == self._sorted_ids[:-1]).any())):
                raise L.StarGCNError("CatalogueHead: item_ids have to be all different and not negative")

    def scores(self, user_rows, residual=None, out_dtype=torch.float32):
        """(users, items) scores."""
        user_rows = user_rows.detach()
        if self.norm_weight is not None:
            codes, scale, _ = ops.rms_norm_i8(user_rows, self.norm_weight, residual=residual, eps=self.eps)
        elif residual is not None:
            raise L.StarGCNError("CatalogueHead: a residual needs norm_weight")
        else:
            codes, scale = ops.quantize_rows(user_rows)
        return ops.gemm_i8(codes, scale, self.codes, self.scale, bias=self.bias, out_dtype=out_dtype)

    def _rows_of(self, ids):
        """The items' rows; -1 for an id that is not of the catalogue."""
        if self.item_ids is None or not self.items or ids.is_floating_point() or ids.dtype == torch.bool:
            return ids
        ids = ids.long()
        at = torch.searchsorted(self._sorted_ids, ids).clamp_(max=self.items - 1)
        return torch.where(self._sorted_ids[at] == ids, self._sorted_rows[at], torch.full_like(at, -1))

    def draw(self, user_rows, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, residual=None, seen=None):
        """One item a user row -> (ids int32 or of item_ids' type, prob fp32), see ops.sample_rows.  seen: (rows of
        user_rows, item ids) index pair of what is not to be drawn, e.g. the items that a user has rated (a pair outside the scores, such as
        padding of -1 or an item that is not in the catalogue, names nothing); a user who has seen everything gets id -1."""
        s = self.scores(user_rows, residual=residual)
        if seen is not None:
            rows, items = (t.to(s.device) for t in seen)
            _mask_pairs(s, rows, self._rows_of(items))
        ids, prob = ops.sample_rows(s, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        if self.item_ids is not None:
            named = self.item_ids[ids.clamp(min=0).long()] if self.items else ids.to(self.item_ids.dtype)
            ids = torch.where(ids >= 0, named, torch.full_like(named, -1))
        return ids, prob
