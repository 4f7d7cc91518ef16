"""A stack of Dense layers for several experts at once: trained with dropout, served in 8-bit integers.

The reference trains a family of Dense stacks one member at a time -- multipleRegression.py builds, fits and
scores one per WRF variable (:28-45, :533-550), each a chain of ``keras.layers.Dense`` (:280-284).  Here
the rows of all members (variables, regions, stations: the experts) go through one launch per layer,
sorted by expert; how many rows each has is known on the device only.

forward : h_0 = x,  h_l = dropout(relu(W_l[g] h_{l-1} + b_l[g])),  the last layer linear and without dropout
backward: g_L = dL/dh_L, then for l = L..1
              (dW_l, db_l) = weight/bias gradients of every expert (h_{l-1}, g_l)
              g_{l-1}      = mask_{l-1} * W_l[g]^T g_l
h_l is positive exactly where the ReLU passed and dropout kept, so it is the ReLU mask of the backward store; the
dropout mask itself is drawn again, never stored.  The gradients land in ONE flat buffer, ready for a single
all-reduce (weather_model_amd.dp).
"""
from __future__ import annotations

import torch

from . import dp, ops


class ExpertStack:
    """weights: (G, N_l, K_l) per layer, biases: (G, N_l); float32, bfloat16 or float16, all alike.  p and seed are
    dropout's (``ops.dropout_forward``); ranks that train together take a seed each, as they draw by the row of their own batch."""

    def __init__(self, weights, biases, p=0.0, seed=0):
        if len(weights) != len(biases) or not weights:
            raise ValueError("one bias per weight, at least one layer")
        self.p, self.seed = ops._dropout_args(p, seed, 0, None)[:2]
        self.w = [ops._req_any(weights[0], "weight")]
        self.w += [ops._req_any(w, "weight", self.w[0]) for w in weights[1:]]
        self.b = [ops._req_any(b, "bias", self.w[0]) for b in biases]
        for l, (w, b) in enumerate(zip(self.w, self.b)):
            if w.dim() != 3 or w.shape[0] != self.w[0].shape[0] or tuple(b.shape) != tuple(w.shape[:2]) or \
                    (l and w.shape[2] != self.w[l - 1].shape[1]):
                raise ValueError(f"layer {l}: weight {tuple(w.shape)} and bias {tuple(b.shape)} do not fit")
        # where each layer's dropout last drew, on the device: the replays of a captured step move on as eager steps do.
        # `span` is the most that any step has drawn from there, so that a step goes past what the one before it drew,
        # however many rows that had; a graph replayed between eager steps finds it on the device too.
        self.drawn = torch.arange(len(weights) - 1, device=self.w[0].device, dtype=torch.int64) << 48
        self.span = torch.zeros((1,), device=self.w[0].device, dtype=torch.int64)
        self.h = None
        sizes = [t.numel() for t in self.w + self.b]
        self.flat_grads = torch.zeros((sum(sizes),), device=self.w[0].device, dtype=self.w[0].dtype)
        views = self.flat_grads.split(sizes)
        self.gw = [v.view(w.shape) for v, w in zip(views, self.w)]
        self.gb = [v.view(b.shape) for v, b in zip(views[len(self.w):], self.b)]
        self.codes = None

    def forward(self, x, offsets, train=False):
        """h_L (M, N_L); with ``train`` dropout is drawn and every activation stays for ``backward``."""
        h, L = [x], len(self.w)
        drop = train and L > 1 and self.p > 0
        if drop:
            self.span.clamp_(min=x.shape[0] * max(w.shape[1] for w in self.w[:-1]))
            self.drawn.add_(self.span)
        for l, (w, b) in enumerate(zip(self.w, self.b)):
            y = ops.dense_grouped_forward(h[-1], w, offsets, b, relu=l + 1 < L)
            if drop and l + 1 < L:
                ops.dropout_forward(y, self.p, self.seed, offset=self.drawn[l:l + 1], out=y)
            h.append(y)
        if train:
            self.h, self.offsets, self.dropped = h, offsets, drop
        return h[-1]

    def backward(self, gout):
        """Gradients of every layer from dL/dh_L of the last ``forward(train=True)``.  Returns the flat
        buffer [dW_1..dW_L, db_1..db_L]."""
        if self.h is None:
            raise RuntimeError("ExpertStack.backward: call forward(train=True) first")
        g = gout
        for l in range(len(self.w), 0, -1):
            g, _, _ = ops.dense_grouped_backward(self.h[l - 1], self.w[l - 1], self.offsets, g,
                                                 mask_below=self.h[l - 1] if l > 1 else None, need_gx=l > 1,
                                                 out_w=self.gw[l - 1], out_b=self.gb[l - 1])
            if l > 1 and self.dropped:
                ops.dropout_backward(g, self.p, self.seed, offset=self.drawn[l - 2:l - 1], out=g)
        return self.flat_grads

    def step_grads(self, x, offsets, gout):
        """forward + backward + (N > 1) the one gradient all-reduce of data parallelism."""
        self.forward(x, offsets, train=True)
        self.backward(gout)
        dp.reduce_grads_(self.flat_grads)
        return self.flat_grads

    def quantize(self):
        """Codes and scales of the present weights, and the present biases, for ``predict``; later changes in place do not
        reach them."""
        self.codes = []
        for w, b in zip(self.w, self.b):
            q, s = ops.quantize_rows(w.reshape(-1, w.shape[2]))
            self.codes.append((q.view(w.shape), s.view(w.shape[:2]), b.to(torch.float32, copy=True)))
        return self

    def predict(self, x, offsets):
        """``forward`` in 8-bit integers, on the codes of the last ``quantize``."""
        if self.codes is None:
            raise RuntimeError("ExpertStack.predict: call quantize() first")
        for l, (q, s, b) in enumerate(self.codes):
            x = ops.dense_i8(x, q, s, b, relu=l + 1 < len(self.codes), offsets=offsets)
        return x
