"""Backward passes made of kernels, which autograd cannot differentiate."""
import functools

import torch


class _Refused(torch.autograd.Function):
    """The first `count` tensors as results of all of them; asked for a derivative, it says why there is none."""

    @staticmethod
    def forward(ctx, name, count, *tensors):
        ctx.name = name
        return tuple(t.detach() for t in tensors[:count])

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("%s cannot be differentiated twice: its backward pass is made of kernels" % ctx.name)


def _leaves(node):
    """What the graph behind a node ends in."""
    todo, seen, leaves = [node], {node}, []
    while todo:
        for below, _ in todo.pop().next_functions:
            if below is not None and below not in seen:
                seen.add(below)
                todo.append(below)
                leaves += [below.variable] if hasattr(below, "variable") else []
    return leaves


def first_order(backward):
    """A Function's backward whose results depend on its inputs in ways that autograd does not see: with create_graph their derivative is an error.  (Unmarked they
    count as constants, and a second derivative leaves their terms out in silence.)  A gradient that is passed on as it arrived stays what it is."""
    @functools.wraps(backward)
    def run(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        inputs = [t for t in (*grads, *ctx.saved_tensors, *_leaves(ctx)) if t is not None and t.requires_grad]
        with torch.no_grad():
            outs = backward(ctx, *grads)
        results = list(outs) if isinstance(outs, tuple) else [outs]
        made = [i for i, v in enumerate(results) if v is not None and not any(v is g for g in grads)]
        if made:
            for i, v in zip(made, _Refused.apply(backward.__qualname__.split(".")[0], len(made), *[results[i] for i in made], *inputs)):
                results[i] = v
        return tuple(results) if isinstance(outs, tuple) else results[0]
    return run
