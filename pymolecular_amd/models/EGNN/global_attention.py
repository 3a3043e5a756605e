"""E_GCL layers alternating with attention over all nodes of each graph.

The message layers of ``egnn_clean.py`` reach a node's neighbours; a network
that also has to see the whole molecule, chain or system alternates them with
attention inside the graph, each followed by "add and normalise", and reads a
graph out with a learned query.  No counterpart in the reference.  The graphs
of a batch lie back to back: graph b holds the nodes seg_ptr[b] ..
seg_ptr[b + 1] - 1 (int32, as in :mod:`pymolecular_amd.graph_build`).
"""
from __future__ import annotations

import torch
from torch import nn

from ...layer_norm import layer_norm
from ...node_update import dense
from ...segment_attention import segment_attention, segment_attention_qkv
from .egnn_clean import E_GCL, _csr_cache

__all__ = ["GlobalAttention", "GraphReadout", "EGNNGlobal"]


def _head_dim(hidden_nf, heads, kv_heads):
    if heads < 1 or hidden_nf % heads or kv_heads < 1 or heads % kv_heads:
        raise ValueError(f"hidden_nf {hidden_nf} needs a number of heads that divides it, and heads {heads} a number of "
                         f"kv_heads that divides them (got {kv_heads})")
    return hidden_nf // heads


class GlobalAttention(nn.Module):
    """Attention of every node over the nodes of its graph; one projection makes queries, keys and values, which are
    read where they lie."""

    def __init__(self, hidden_nf, heads=4, kv_heads=None):
        super().__init__()
        self.heads, self.kv_heads = heads, heads if kv_heads is None else kv_heads
        d = _head_dim(hidden_nf, heads, self.kv_heads)
        self.qkv = nn.Linear(hidden_nf, (heads + 2 * self.kv_heads) * d)
        self.out = nn.Linear(hidden_nf, hidden_nf)

    def forward(self, h, seg_ptr, key_mask=None):
        qkv = dense(h, self.qkv).view(h.shape[0], self.heads + 2 * self.kv_heads, -1)
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
    of the attention (they keep their messages)."""

    def __init__(self, in_node_nf, hidden_nf, out_nf, in_edge_nf=0, device='cpu', act_fn=nn.SiLU(), n_layers=4, heads=4,
                 kv_heads=None, eps=1e-5):
        super().__init__()
        self.n_layers, self.eps = n_layers, eps
        self.embedding_in = nn.Linear(in_node_nf, hidden_nf)
        self.embedding_out = nn.Linear(hidden_nf, out_nf)
        self.readout = GraphReadout(hidden_nf, heads, kv_heads)
        for i in range(n_layers):
            self.add_module("gcl_%d" % i, E_GCL(hidden_nf, hidden_nf, hidden_nf, edges_in_d=in_edge_nf, act_fn=act_fn,
                                                residual=False))
            self.add_module("att_%d" % i, GlobalAttention(hidden_nf, heads, kv_heads))
            for name in ("gcl_norm_%d", "att_norm_%d"):
                self.add_module(name % i, nn.LayerNorm(hidden_nf, eps=eps))
        self.to(device)

    def _add_norm(self, update, h, norm):
        return layer_norm(update, norm.weight, norm.bias, self.eps, residual=h)[0]

    def forward(self, h, x, edges, edge_attr, seg_ptr, node_mask=None):
        m = self._modules
        h = dense(h, self.embedding_in)
        row, col = edges
        csr = _csr_cache.get(row, col, h.shape[0])   # one CSR for all layers, cached per edge tensor
        for i in range(self.n_layers):
            u, x, _ = m["gcl_%d" % i](h, edges, x, edge_attr=edge_attr, csr=csr)
            h = self._add_norm(u, h, m["gcl_norm_%d" % i])
            h = self._add_norm(m["att_%d" % i](h, seg_ptr, node_mask), h, m["att_norm_%d" % i])
        return dense(self.readout(h, seg_ptr, node_mask), self.embedding_out), h, x
