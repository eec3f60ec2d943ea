"""The accepted drafted tokens' rows to the front of their range (pdattn_accept_kv).

CPU: the restatement (oracle.accept_kv) against a gather by fancy indexing, with planted mistakes; refusals. GPU: the
caches byte for byte, invalid lists counted and their sequences left alone.
"""
import numpy as np
import pytest

import oracle
import pdattn
from pdattn import inputs


def _batch(ctx, new, Hkv, seed):
    bt = inputs.make_batch([c + n for c, n in zip(ctx, new)], Hkv, Hkv, seed)
    return bt, np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def _lists(new, rng, most=9):
    out = [np.sort(rng.choice(n, min(n, int(rng.integers(0, most))), replace=False)) if n else np.zeros(0, int) for n in new]
    return np.concatenate([[0], np.cumsum([len(x) for x in out])]).astype(np.int32), np.concatenate(out + [np.zeros(0, int)]).astype(np.int32)


def _gathered(bt, q_indptr, aip, acc):
    """All rows read first, then written."""
    kc, vc = bt.k.copy(), bt.v.copy()
    for b in range(bt.B):
        a = acc[aip[b]:aip[b + 1]]
        ctx = bt.lens[b] - int(q_indptr[b + 1] - q_indptr[b])
        pages = bt.indices[bt.indptr[b]:bt.indptr[b + 1]]
        src, dst = ctx + a, ctx + np.arange(len(a))
        for c, old in ((kc, bt.k), (vc, bt.v)):
            c[pages[dst // 16], dst % 16] = old[pages[src // 16], src % 16]
    return kc, vc


CASES = [([37, 16, 1, 0], [9, 40, 1, 33]), ([300], [64]), ([15, 14], [2, 20])]


def _agrees(ctx, new, seed, fault="none"):
    bt, qi = _batch(ctx, new, 2, seed)
    aip, acc = _lists(new, np.random.default_rng(seed))
    kc, vc, bad = oracle.accept_kv(bt.k, bt.v, bt.indptr, bt.indices, bt.last, qi, aip, acc, fault)
    rk, rv = _gathered(bt, qi, aip, acc)
    return bad == 0 and np.array_equal(kc, rk) and np.array_equal(vc, rv)


@pytest.mark.parametrize("seed", range(5))
@pytest.mark.parametrize("case", CASES)
def test_restatement_is_a_gather(case, seed):
    assert _agrees(*case, seed)


@pytest.mark.parametrize("fault", [f for f in oracle.ACCEPT_FAULTS if f != "none"])
def test_planted_fault_is_caught(fault):
    assert not all(_agrees(*c, s, fault) for c in CASES for s in range(5))


@pytest.mark.parametrize("change", [{0: None}, {1: None}, {2: None}, {3: None}, {4: None}, {5: None}, {6: None}, {7: None},
                                    {0: (1 << 20) + 8}, {1: (1 << 20) + 2}, {8: -1}, {9: 0}, {9: -2}])
def test_refusals(change):
    args = [1 << 20] * 8 + [2, 2]
    for i, x in change.items():
        args[i] = x
    with pytest.raises(pdattn.PdattnError) as e:
        pdattn.accept_kv(*args)
    assert e.value.status == 1


def test_no_sequences():
    pdattn.accept_kv(*[1 << 20] * 8, 0, 2)


def _gpu_case(ctx, new, Hkv, aip, acc, seed, tag):
    import torch
    from _gpu import DeviceBatch, device
    bt, qi = _batch(ctx, new, Hkv, seed)
    db = DeviceBatch(bt)
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(device())  # noqa: E731
    dq, da, dl = put(qi), put(aip), put(acc if len(acc) else np.zeros(1))
    bad = torch.zeros(1, dtype=torch.int32, device=device())
    print(f"accept {tag}", flush=True)
    pdattn.accept_kv(db.k, db.v, db.indptr, db.indices, db.last, dq, da, dl, bt.B, Hkv, bad)
    torch.cuda.synchronize()
    kc, vc, nbad = oracle.accept_kv(bt.k, bt.v, bt.indptr, bt.indices, bt.last, qi, aip, acc)
    assert int(bad.item()) == nbad
    assert np.array_equal(db.k.cpu().numpy().view(np.uint16), kc.view(np.uint16))
    assert np.array_equal(db.v.cpu().numpy().view(np.uint16), vc.view(np.uint16))
    return nbad


@pytest.mark.gpu
@pytest.mark.parametrize("Hkv", [1, 2, 3, 8, 32])
@pytest.mark.parametrize("most", [2, 9, 200])
def test_paths(Hkv, most):
    rng = np.random.default_rng(Hkv + most)
    ctx, new = [37, 16, 1, 0, 250], [9, 40, 1, 133, 64]
    _gpu_case(ctx, new, Hkv, *_lists(new, rng, most), seed=Hkv, tag=f"Hkv={Hkv} most={most}")


@pytest.mark.gpu
def test_all_and_nearly_all_accepted():
    """Lists longer than a thread's rows in flight: the whole draft, all but its first token, every second."""
    new = [200, 200, 201, 8, 9]
    lists = [np.arange(200), np.arange(1, 200), np.arange(0, 201, 2), np.arange(8), np.arange(1, 9)]
    aip = np.concatenate([[0], np.cumsum([len(x) for x in lists])])
    _gpu_case([3, 30, 17, 16, 15], new, 4, aip, np.concatenate(lists), seed=3, tag="long lists")


@pytest.mark.gpu
def test_invalid_lists_leave_their_sequence_alone():
    new = [5, 5, 5, 5, 5, 80, 80]
    lists = [[0, 5], [-1, 2], [2, 2], [3, 1], [1, 4], list(range(10, 79)) + [78], [70, 79]]
    aip = np.concatenate([[0], np.cumsum([len(x) for x in lists])])
    assert _gpu_case([20] * 7, new, 2, aip, np.concatenate(lists), seed=5, tag="invalid") == 5


@pytest.mark.gpu
def test_many_sequences():
    rng = np.random.default_rng(6)
    ctx, new = rng.integers(0, 30, 700).tolist(), rng.integers(0, 12, 700).tolist()
    _gpu_case(ctx, new, 2, *_lists(new, rng, 6), seed=7, tag="700 sequences")
