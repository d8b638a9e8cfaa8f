"""Norms of queries and keys, head by head, with the rotation and the append, against their definition in float64."""

from __future__ import annotations

import math

import pytest
import torch

from klcquant_amd import ops

pytestmark = pytest.mark.gpu
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def normed(x, weight, eps):
    if weight is None:
        return x.double()
    x = x.double()
    return x / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + eps) * weight.double()


def rotated(x, cos, sin, positions):
    """The rotation, and the sum of its terms' sizes."""
    a, b = x.chunk(2, dim=-1)
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
    return (torch.cat((a * c - b * s, b * c + a * s), dim=-1),
            torch.cat(((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()), dim=-1))


def assert_near(got, want, size, dtype):
    """Float32: the factor's rounding and its two products, 3 x 2^-24 of each term, the product and the sum of the
    rotation, 2 x 2^-24; then one rounding to the type, and of subnormals half a step of the smallest."""
    eps = torch.finfo(dtype).eps / 2
    off = 6 * 2.0 ** -24 * size
    off = off + eps * (want.abs() + off) + torch.finfo(dtype).tiny * eps
    assert ((got.double() - want).abs() <= off).all(), float(((got.double() - want).abs() / off).max())


def inputs(gpu, tokens, heads, kv, dim, fused=False, std=3.0):
    g = torch.Generator(device=gpu).manual_seed(dim + tokens)
    x = (torch.randn((tokens, heads + 2 * kv, dim), device=gpu, generator=g) * std).bfloat16()
    q, k, v = x.split((heads, kv, kv), dim=1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    angle = torch.rand((500, dim // 2), device=gpu, generator=g) * 6.3
    weights = [(1 + 0.3 * torch.randn(dim, device=gpu, generator=g)).bfloat16() for _ in range(2)]
    return q, k, v, angle.cos().bfloat16(), angle.sin().bfloat16(), *weights


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("tokens,heads,kv,dim,fused", [(1, 64, 8, 64, False), (77, 64, 8, 64, True), (33, 7, 1, 80, False),
                                                       (300, 3, 3, 8, True), (5, 8, 2, 128, False), (19, 4, 1, 24, True),
                                                       (40, 6, 2, 96, True), (11, 5, 5, 48, False), (9, 2, 1, 120, True),
                                                       (3, 4, 2, 16, False), (3, 4, 2, 56, False)])
@pytest.mark.parametrize("which", ["both", "q", "k"])
def test_norms(gpu, dtype, tokens, heads, kv, dim, fused, which):
    q, k, v, cos, sin, wq, wk = inputs(gpu, tokens, heads, kv, dim, fused)
    wq, wk = (wq if which != "k" else None), (wk if which != "q" else None)
    page, n_pages, eps = 16, 3 + tokens // 8, 1e-5
    g = torch.Generator().manual_seed(tokens)
    positions = torch.randint(0, 500, (tokens,), generator=g).to(gpu)
    slots = torch.randperm(n_pages * page, generator=g)[:tokens].to(gpu)
    drop = tokens // 3
    where = slots.clone()
    where[:drop] = torch.tensor([-1, n_pages * page, -2 ** 31, 2 ** 31 - 1], device=gpu)[torch.arange(drop, device=gpu) % 4]
    pools = [torch.full((n_pages, page, kv, dim), 9.0, dtype=DTYPES[dtype], device=gpu) for _ in range(2)]
    rq, rk = ops.paged_append(q, k, v, cos, sin, positions.int(), where.int(), *pools, q_norm=wq, k_norm=wk, eps=eps)
    (want_q, size_q), (want_k, size_k) = (rotated(normed(x, w, eps), cos, sin, positions) for x, w in ((q, wq), (k, wk)))
    assert_near(rq, want_q, size_q, torch.bfloat16)
    assert_near(rk, want_k, size_k, torch.bfloat16)
    flat_k, flat_v = (p.view(-1, kv, dim) for p in pools)
    assert_near(flat_k[slots[drop:]], want_k[drop:], size_k[drop:], DTYPES[dtype])
    assert torch.equal(flat_v[slots[drop:]], v[drop:].float().to(DTYPES[dtype]))
    rest = torch.ones(n_pages * page, dtype=torch.bool, device=gpu)
    rest[slots[drop:]] = False
    assert (flat_k[rest] == 9).all() and (flat_v[rest] == 9).all()
    again, none = ops.paged_append(q, k, v, cos, sin, positions.int(), where.int(), *pools, want_keys=False, q_norm=wq,
                                   k_norm=wk, eps=eps)
    assert torch.equal(again, rq) and none is None
    if which != "both":  # what is not normalised is what it was
        plain = ops.paged_append(q, k, v, cos, sin, positions.int(), where.int(), *pools)
        assert torch.equal(plain[which == "q"], (rq, rk)[which == "q"])


@pytest.mark.parametrize("dim", [64, 128, 24])
def test_sizes_of_all_kinds(gpu, dim):
    """Squares that overflow or vanish in float32, zeros, subnormals, one infinity and one NaN."""
    q, k, v, cos, sin, wq, wk = inputs(gpu, 8, 4, 2, dim)
    for i, factor in enumerate((2.0 ** 100, 2.0 ** -100, 0.0, 2.0 ** -130, 2.0 ** 60)):
        q[i], k[i] = q[i] * factor, k[i] * factor
    q[5, 0, 3], q[6, 1, dim - 1] = math.inf, math.nan
    positions = torch.arange(8, device=gpu)
    pools = [torch.zeros((1, 16, 2, dim), dtype=torch.bfloat16, device=gpu) for _ in range(2)]
    for eps in (1e-6, 0.0):
        rq, rk = ops.paged_append(q, k, v, cos, sin, positions.int(), positions.int(), *pools, q_norm=wq, k_norm=wk, eps=eps)
        for got, x, w in ((rq, q, wq), (rk, k, wk)):
            want, size = rotated(normed(x, w, eps), cos, sin, positions)
            assert torch.equal(got.isnan(), want.isnan())
            fine = torch.isfinite(want)
            assert_near(got[fine], want[fine], size[fine], torch.bfloat16)


def test_positions_and_no_tokens(gpu):
    q, k, v, cos, sin, wq, wk = inputs(gpu, 3, 4, 2, 64)
    pools = [torch.zeros((1, 16, 2, 64), dtype=torch.float16, device=gpu) for _ in range(2)]
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    rq, rk = ops.paged_append(q, k, v, cos, sin, i(499, 500, -1), i(0, 1, 2), *pools, q_norm=wq, k_norm=wk)
    assert torch.isfinite(rq[0]).all() and rq[1:].isnan().all() and rk[1:].isnan().all()
    assert pools[0][0, 1:3].isnan().all() and torch.equal(pools[1][0, :3], v.to(torch.float16))
    rq, rk = ops.paged_append(q[:0], k[:0], v[:0], cos, sin, i(), i(), *pools, q_norm=wq, k_norm=wk)
    assert rq.shape == (0, 4, 64) and rk.shape == (0, 2, 64)


def test_captured_and_replayed(gpu):
    q, k, v, cos, sin, wq, wk = inputs(gpu, 20, 4, 2, 64)
    at = torch.arange(20, dtype=torch.int32, device=gpu)
    pools, others = ([torch.zeros((2, 16, 2, 64), dtype=torch.float16, device=gpu) for _ in range(2)] for _ in range(2))
    ops.paged_append(q, k, v, cos, sin, at, at, *pools, q_norm=wq, k_norm=wk)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rq, rk = ops.paged_append(q, k, v, cos, sin, at, at, *pools, q_norm=wq, k_norm=wk)
    for _ in range(3):
        q.copy_(torch.randn_like(q))
        k.copy_(torch.randn_like(k))
        graph.replay()
        torch.cuda.synchronize()
        want = ops.paged_append(q, k, v, cos, sin, at, at, *others, q_norm=wq, k_norm=wk)
        assert torch.equal(rq, want[0]) and torch.equal(rk, want[1]) and torch.equal(pools[0], others[0])
