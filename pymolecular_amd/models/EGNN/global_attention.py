"""E_GCL layers alternating with attention over all nodes of each graph.

The message layers of ``egnn_clean.py`` reach a node's neighbours; a network
that also has to see the whole molecule, chain or system alternates them with
attention inside the graph, each followed by "add and normalise", and reads a
graph out with a learned query.  No counterpart in the reference.  The graphs
of a batch lie back to back: graph b holds the nodes seg_ptr[b] ..
seg_ptr[b + 1] - 1 (int32, as in :mod:`pymolecular_amd.graph_build`).

Nodes may come as types instead of features (``n_types``: a table of one vector
a type), queries and keys of the attention may be normed and turned by the
nodes' positions along a chain (``qk_norm``), and training may drop values in
front of each residual sum (``dropout``).
"""
from __future__ import annotations

import torch
from torch import nn

from ...dropout import Dropout, dropout
from ...embedding import embedding
from ...layer_norm import layer_norm, layer_norm_dropout
from ...node_update import dense
from ...qk_norm_rotary import MAX_HEAD_DIM, qk_norm_rotary_attention
from ...segment_attention import segment_attention, segment_attention_qkv
from .egnn_clean import E_GCL, _csr_cache

__all__ = ["TypeEmbedding", "GlobalAttention", "GraphReadout", "EGNNGlobal"]


def _head_dim(hidden_nf, heads, kv_heads):
    if heads < 1 or hidden_nf % heads or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"hidden_nf {hidden_nf} needs a number of heads that divides it, and heads {heads} a number of "
                         f"kv_heads that divides them (got {kv_heads})")
    return hidden_nf // heads


class TypeEmbedding(nn.Module):
    """One vector a node type: hidden_nf ** 0.5 times a row of a table whose rows have length of about 1.  ``dtype``: of
    the vectors (None: the table's; bfloat16 beside a float32 table keeps its gradients in float32).  The row
    ``padding_type`` gets no gradient.  A type outside the table has a vector of zeros and no gradient; it is not an error,
    which would have to wait for the device."""

    def __init__(self, n_types, hidden_nf, padding_type=None, dtype=None):
        super().__init__()
        self.weight = nn.Parameter(torch.randn(n_types, hidden_nf) * hidden_nf ** -0.5)
        self.scale, self.padding_type, self.dtype = hidden_nf ** 0.5, padding_type, dtype

    def forward(self, types):
        return embedding(types, self.weight, self.scale, self.padding_type, dtype=self.dtype)


class GlobalAttention(nn.Module):
    """Attention of every node over the nodes of its graph; one projection makes queries, keys and values, which are
    read where they lie.  ``qk_norm``: every head of queries and keys is normed, with a weight for each, and turned by
    ``positions`` (N,) where they are given."""

    def __init__(self, hidden_nf, heads=4, kv_heads=None, qk_norm=False, rotary_base=10000.0):
        super().__init__()
        self.heads, self.kv_heads = heads, heads if kv_heads is None else kv_heads
        d = _head_dim(hidden_nf, heads, self.kv_heads)
        if qk_norm and (d % 2 or d > MAX_HEAD_DIM):
            raise ValueError(f"qk_norm needs heads of an even width up to {MAX_HEAD_DIM} (hidden_nf {hidden_nf} / heads "
                             f"{heads} is {d})")
        self.qkv = nn.Linear(hidden_nf, (heads + 2 * self.kv_heads) * d)
        self.out = nn.Linear(hidden_nf, hidden_nf)
        self.qk_norm, self.rotary_base = qk_norm, rotary_base
        if qk_norm:
            self.q_weight, self.k_weight = nn.Parameter(torch.ones(d)), nn.Parameter(torch.ones(d))

    def forward(self, h, seg_ptr, key_mask=None, positions=None):
        qkv = dense(h, self.qkv).view(h.shape[0], self.heads + 2 * self.kv_heads, -1)
        if self.qk_norm:
            a = qk_norm_rotary_attention(qkv, self.heads, seg_ptr, self.q_weight, self.k_weight, positions, key_mask,
                                         base=self.rotary_base)
        elif positions is not None:
            raise ValueError("positions turn normed queries and keys: the attention needs qk_norm")
        else:
            a = segment_attention_qkv(qkv, self.heads, seg_ptr, key_mask)
        return dense(a.reshape(h.shape[0], -1), self.out)


class GraphReadout(nn.Module):
    """One vector a graph: a learned query attends the nodes of each graph (0 where none is left)."""

    def __init__(self, hidden_nf, heads=4, kv_heads=None):
        super().__init__()
        self.heads, self.kv_heads = heads, heads if kv_heads is None else kv_heads
        d = _head_dim(hidden_nf, heads, self.kv_heads)
        self.query = nn.Parameter(torch.randn(heads, d))
        self.kv = nn.Linear(hidden_nf, 2 * self.kv_heads * d)

    def forward(self, h, seg_ptr, key_mask=None):
        n_graphs = seg_ptr.numel() - 1
        kv = dense(h, self.kv).view(h.shape[0], 2 * self.kv_heads, -1)
        q = self.query.to(h.dtype).expand(n_graphs, *self.query.shape)
        q_ptr = torch.arange(n_graphs + 1, dtype=torch.int32, device=h.device)
        out = segment_attention(q, kv[:, :self.kv_heads], kv[:, self.kv_heads:], q_ptr, seg_ptr, key_mask)
        return out.reshape(n_graphs, -1)


class EGNNGlobal(nn.Module):
    """embedding_in, ``n_layers`` x (E_GCL, add and normalise, GlobalAttention, add and normalise), GraphReadout,
    embedding_out.  ``forward`` returns ``(graph outputs (n_graphs, out_nf), h, x)``; ``node_mask`` (N,) leaves nodes out
    of the attention (they keep their messages).

    ``n_types``: ``h`` holds a type (N,) of each node instead of features (``in_node_nf`` is 0 then), and ``node_dtype`` is
    the dtype of their vectors (None: the parameters').  ``qk_norm``, ``rotary_base``: see :class:`GlobalAttention`;
    ``forward`` takes ``positions`` then.  ``dropout``: the probability, in training, with which a value of the embedding
    and of each update is dropped in front of its residual sum.  Its masks come from the buffer ``dropout_state`` (seed and
    offset), whose offset each such pass advances on the device, so a captured pass draws anew on every replay.  Replicas of
    a network want a seed each (:meth:`seed_dropout`; and no broadcast of buffers), and a pass that is made again for its
    backward has to start from the same state."""

    def __init__(self, in_node_nf, hidden_nf, out_nf, in_edge_nf=0, device='cpu', act_fn=nn.SiLU(), n_layers=4, heads=4,
                 kv_heads=None, eps=1e-5, n_types=None, node_dtype=None, qk_norm=False, rotary_base=10000.0, dropout=0.0):
        super().__init__()
        if n_types is not None and in_node_nf:
            raise ValueError(f"nodes are types or features: n_types {n_types} needs an in_node_nf of 0 (got {in_node_nf})")
        if not 0.0 <= dropout < 1.0:
            raise ValueError(f"the probability of a dropout must be 0 or more and below 1 (got {dropout})")
        self.n_layers, self.eps, self.dropout = n_layers, eps, dropout
        if n_types is None:
            self.embedding_in = nn.Linear(in_node_nf, hidden_nf)
        else:
            self.embedding_in = TypeEmbedding(n_types, hidden_nf, dtype=node_dtype)
        self.embedding_out = nn.Linear(hidden_nf, out_nf)
        self.readout = GraphReadout(hidden_nf, heads, kv_heads)
        for i in range(n_layers):
            self.add_module("gcl_%d" % i, E_GCL(hidden_nf, hidden_nf, hidden_nf, edges_in_d=in_edge_nf, act_fn=act_fn,
                                                residual=False))
            self.add_module("att_%d" % i, GlobalAttention(hidden_nf, heads, kv_heads, qk_norm, rotary_base))
            for name in ("gcl_norm_%d", "att_norm_%d"):
                self.add_module(name % i, nn.LayerNorm(hidden_nf, eps=eps))
        if dropout:
            self.register_buffer("dropout_state", torch.stack([torch.randint(1 << 62, ()), torch.zeros((), dtype=torch.int64)]))
        self.to(device)

    def seed_dropout(self, seed, offset=0):
        """Where the masks go on from."""
        self.dropout_state.copy_(torch.tensor([seed, offset], dtype=torch.int64))

    def _add_norm(self, update, h, norm, drop=None):
        if drop is not None:
            return layer_norm_dropout(update, h, drop, norm.weight, norm.bias, self.eps)[0]
        return layer_norm(update, norm.weight, norm.bias, self.eps, residual=h)[0]

    def forward(self, h, x, edges, edge_attr, seg_ptr, node_mask=None, positions=None):
        m = self._modules
        h = self.embedding_in(h) if isinstance(self.embedding_in, TypeEmbedding) else dense(h, self.embedding_in)
        drop = lambda site: None  # noqa: E731
        if self.dropout and self.training:
            self.dropout_state[1] += 2 * self.n_layers + 1   # one for each site
            rng = self.dropout_state.clone()
            drop = lambda site: Dropout(self.dropout, rng, site)  # noqa: E731
            h = dropout(h, *drop(0)[:2])
        row, col = edges
        csr = _csr_cache.get(row, col, h.shape[0])   # one CSR for all layers, cached per edge tensor
        for i in range(self.n_layers):
            u, x, _ = m["gcl_%d" % i](h, edges, x, edge_attr=edge_attr, csr=csr)
            h = self._add_norm(u, h, m["gcl_norm_%d" % i], drop(2 * i + 1))
            h = self._add_norm(m["att_%d" % i](h, seg_ptr, node_mask, positions), h, m["att_norm_%d" % i], drop(2 * i + 2))
        return dense(self.readout(h, seg_ptr, node_mask), self.embedding_out), h, x
