"""Causal training: NaN or infinity in one row reaches the gradients that depend on it and no others.

The reference is the same call with that row (or value) at zero: what does not
depend on it has the same bits.  Query r of a sequence sees keys j ≤ r + lk − lq:
dq_i depends on query i and the keys that it sees, dk_j and dv_j on the queries
that see key j; dv not on v, and its columns each on the same column of grad_out.
"""
import pytest
import torch

from test_packed_attention_gpu import TYPES, _plan, _qkv

pytestmark = pytest.mark.gpu
COLUMN = 5
CASES = [([300], [300], 2, 2, 64), ([700, 150, 64, 100], [700, 150, 64, 100], 4, 2, 128), ([1000, 900], [1000, 900], 6, 3, 80),
         ([40, 9], [1500, 70], 4, 1, 64), ([300, 140], [200, 60], 4, 4, 64), ([3000], [3000], 8, 1, 64)]


def _grads(q, k, v, do, plan):
    from vision_rs_b200 import packed
    o, lse = packed.packed_attention_forward(q, k, v, plan)
    return packed.packed_attention_backward(do, q, k, v, o, lse, plan)


def _spots(lq, lk):
    """A row of each sequence (late, early, one that sees nothing) as queries and as keys."""
    for late in (True, False):
        qs, ks = [], []
        for a, b in zip(lq, lk):
            qs.append(a - 1 - min(a - 1, 37) if late else min(a - 1, 70))
            ks.append(b - min(b, 41) if late else min(b - 1, 3))
        yield qs, ks


def _sets(lq, lk, rows, keys):
    """Per token: queries that are the row itself, keys that the row sees, queries that see the key."""
    own, seen, sees = [], [], []
    for a, b, r, j in zip(lq, lk, rows, keys):
        own += [i == r for i in range(a)]
        seen += [m <= r + b - a for m in range(b)]
        sees += [i >= j - (b - a) for i in range(a)]
    return (torch.tensor(x) for x in (own, seen, sees))


def _put(t, at, lengths, value, column):
    t, first = t.clone(), 0
    for n, i in zip(lengths, at):
        t[first + i, :, slice(None) if column is None else column] = value
        first += n
    return t


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lq,lk,H,Hk,D", CASES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_queries_and_their_gradients(cuda, dt, lq, lk, H, Hk, D, bad):
    q, k, v = _qkv(cuda, dt, lq, lk, H, Hk, D, seed=3)
    do = torch.randn(q.shape, generator=torch.Generator().manual_seed(4)).to(cuda, dt)
    plan = _plan(lq, lk, H, Hk, D, True, training=True)
    for rows, keys in _spots(lq, lk):
        own, seen, _ = _sets(lq, lk, rows, keys)
        for column in (None, COLUMN):
            got = _grads(_put(q, rows, lq, bad, column), k, v, do, plan)
            ref = _grads(_put(q, rows, lq, 0, column), k, v, do, plan)
            assert torch.equal(got[0][~own], ref[0][~own])
            for g, r in zip(got[1:], ref[1:]):
                assert torch.equal(g[~seen], r[~seen])
                if bad != bad:
                    assert g[seen].isnan().all()
            got = _grads(q, k, v, _put(do, rows, lq, bad, column), plan)
            ref = _grads(q, k, v, _put(do, rows, lq, 0, column), plan)
            assert torch.equal(got[0][~own], ref[0][~own])
            for g, r in zip(got[1:], ref[1:]):
                assert torch.equal(g[~seen], r[~seen])
            assert not got[1][seen].isfinite().any()
            hit = slice(None) if column is None else column
            at = got[2][seen][..., hit]
            assert (at.isnan() if bad != bad else at == bad).all()
            if column is not None:
                rest = [c for c in range(D) if c != column]
                assert torch.equal(got[2][..., rest], ref[2][..., rest])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lq,lk,H,Hk,D", CASES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_keys_and_values(cuda, dt, lq, lk, H, Hk, D, bad):
    q, k, v = _qkv(cuda, dt, lq, lk, H, Hk, D, seed=5)
    do = torch.randn(q.shape, generator=torch.Generator().manual_seed(6)).to(cuda, dt)
    plan = _plan(lq, lk, H, Hk, D, True, training=True)
    for rows, keys in _spots(lq, lk):
        _, _, sees = _sets(lq, lk, rows, keys)
        for column in (None, COLUMN):
            got = _grads(q, _put(k, keys, lk, bad, column), v, do, plan)
            ref = _grads(q, _put(k, keys, lk, 0, column), v, do, plan)
            assert torch.equal(got[0][~sees], ref[0][~sees])
            if bad != bad:
                assert got[0][sees].isnan().all()
            got = _grads(q, k, _put(v, keys, lk, bad, column), do, plan)
            ref = _grads(q, k, _put(v, keys, lk, 0, column), do, plan)
            assert torch.equal(got[0][~sees], ref[0][~sees]) and torch.equal(got[2], ref[2])
            if bad != bad:
                assert got[0][sees].isnan().all()
