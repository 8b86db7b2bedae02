"""Rotary positions at the sizes of training calls: several heads of a token in one thread, which share its angles, and results past the caches.  (Tolerances and the computation in 64 bits are those
of test_rotary_embed_gpu.py.)"""
import pytest
import torch

from test_rotary_embed_gpu import check, frequencies, rnd

pytestmark = pytest.mark.gpu


def variant(s, b, nq, nk, d, turned, interleaved):
    """((pairing, whole pieces, heads of a thread, results past the caches), heads that the last threads lack, rows of workgroups over the heads): the rule of ezl_rotary"""
    turned_slots = (turned + 7) // 8 if interleaved else (turned // 2 + 7) // 8
    slots = turned_slots + (d - turned + 7) // 8
    heads = nq + nk
    items = s * b * heads * slots
    each = 1 if items <= 1 << 16 else 2 if items <= 3 << 17 else 8 if interleaved else 4
    lanes = min((heads + each - 1) // each, 256 // slots)
    whole = turned % (8 if interleaved else 16) == 0
    return (interleaved, whole, each, whole and s * b * heads * d * 2 > 264 << 20), -heads % (each * lanes), -(-heads // (each * lanes))


SHAPES = [  # s, b, nq, nk, d, turned, interleaved
    # one head a thread, and two from 2^16 pieces on
    (64, 1, 8, 8, 128, 128, False), (64, 1, 8, 8, 128, 128, True), (61, 1, 8, 8, 128, 100, False), (61, 1, 8, 8, 128, 100, True),
    (1025, 1, 5, 3, 128, 128, False), (513, 1, 5, 3, 128, 128, True), (701, 3, 5, 2, 64, 36, False), (701, 3, 5, 2, 64, 36, True), (201, 1, 21, 4, 256, 64, False), (129, 2, 12, 5, 256, 224, True),
    # four heads, or of neighbours eight, from 3 * 2^17 on
    (1367, 3, 9, 4, 128, 128, False), (911, 3, 9, 4, 128, 128, True), (2731, 2, 7, 4, 80, 40, False), (2731, 2, 7, 4, 80, 40, True), (3001, 1, 13, 6, 96, 66, False), (3001, 1, 13, 6, 96, 66, True),
    (1031, 1, 11, 3, 256, 256, False), (1031, 1, 11, 3, 256, 256, True), (4001, 1, 17, 2, 64, 32, False), (4001, 1, 17, 2, 64, 24, True),
    # few threads for many heads: workgroups of their own for the rest of them
    (301, 1, 17, 2, 1024, 1024, True), (301, 1, 17, 2, 1024, 1024, False), (301, 1, 17, 2, 1024, 1004, True), (129, 2, 12, 5, 256, 220, True), (801, 1, 17, 2, 1024, 1024, False), (1001, 1, 17, 2, 1024, 1000, False), (157, 1, 19, 2, 1024, 996, False), (41, 1, 5, 2, 2048, 2000, True), (33, 1, 5, 2, 2048, 2048, False),
    # more than the caches hold
    (16411, 1, 33, 33, 128, 128, False), (16411, 1, 33, 33, 128, 128, True), (8209, 2, 40, 26, 128, 64, False), (8209, 2, 40, 26, 128, 48, True), (16411, 1, 33, 33, 128, 100, False),
    (16411, 1, 33, 33, 128, 100, True),
]


def test_the_shapes_reach_every_variant():
    seen = [variant(*s) for s in SHAPES]
    every = {(i, w, n, False) for i in (False, True) for w in (False, True) for n in (1, 2, 8 if i else 4)} | {(i, True, 8 if i else 4, True) for i in (False, True)}
    assert every == {v for v, _, _ in seen}
    assert every - {v for v in every if v[2] == 1} <= {v for v, lacking, _ in seen if lacking}  # (where a thread has several heads: also with some of them missing)
    assert {v[:3] for v, _, rows in seen if rows > 1} >= {v[:3] for v in every if v[2] > 1}


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("s,b,nq,nk,d,turned,interleaved", SHAPES)
def test_forward_and_backward(s, b, nq, nk, d, turned, interleaved, packed):
    from easyllm_amd import functional as F
    print("rotary", s, b, nq, nk, d, turned, interleaved, packed, variant(s, b, nq, nk, d, turned, interleaved), flush=True)
    if packed:  # read out of a projection's result, keys first
        both = rnd(s, b, (nk + nq + 1) * d, seed=1)
        k, q = both[..., d:(1 + nk) * d].unflatten(-1, (nk, d)), both[..., (1 + nk) * d:].unflatten(-1, (nq, d))
    else:
        q, k = rnd(s, b, nq, d, seed=1), rnd(s, b, nk, d, seed=2)
    q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
    inv_freq = frequencies(turned)
    positions = torch.randint(0, 1 << 20, (b, s), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    yq, yk = F.rotary_embed(q, k, inv_freq, positions, interleaved=interleaved, scale=1.25)
    dq, dk = rnd(b, s, nq, d, seed=4).transpose(0, 1) if packed else rnd(s, b, nq, d, seed=4), rnd(s, b, nk, d, seed=5)
    gq, gk = torch.autograd.grad((yq, yk), (q, k), (dq, dk))
    for got, x, back in ((yq, q, False), (yk, k, False), (gq, dq, True), (gk, dk, True)):
        for first in range(0, s, 4096):  # (in 64 bits a part at a time)
            rows = slice(first, first + 4096)
            check(got[rows].detach(), x[rows].detach(), inv_freq, positions[:, rows], interleaved, 1.25, back=back)
