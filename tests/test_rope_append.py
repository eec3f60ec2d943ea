"""Rotary positions with the paged append (pdattn_rope_append_kv, pdattn_rope_frequencies).

CPU: the frequencies against formulas of their own; the restatement (oracle.rope) against complex multiplication,
with planted mistakes; refusals. GPU: q_out, the caches and the count of invalid tokens against the restatement, for
both pairings, every kind of rotary size, far positions, slices of one projection's output, q in place.

Tolerance of a rotated element (u, w) -> u cos a - w sin a, half a step being 2^-11 of fp16 and 2^-24 of fp32: the
angle's fraction of a turn is rounded to 32 bits (2^-25 of half a turn, 2^-23.3 radians), sin and cos to 2 steps of
theirs, their product with scale, each product and the sum once more: 2^-20 scale (|u| + |w|) holds all of it; then the
result's own rounding, 2^-11 of it (2^-25 below fp16's normal range).
"""
import numpy as np
import pytest

import oracle
import pdattn
from pdattn import inputs

SCALINGS = {"plain": pdattn.ROPE_PLAIN, "linear": pdattn.ROPE_LINEAR, "base": pdattn.ROPE_BASE,
            "yarn": pdattn.ROPE_YARN, "wavelength": pdattn.ROPE_WAVELENGTH}


# ---- CPU: frequencies ------------------------------------------------------------------------------

@pytest.mark.parametrize("dims", [2, 4, 20, 64, 96, 128])
@pytest.mark.parametrize("base", [10000.0, 500000.0])
def test_plain_linear_and_base(dims, base):
    i = np.arange(dims // 2)
    plain = np.array([base ** (-2 * x / dims) for x in i])
    f, s = pdattn.rope_frequencies(dims, base)
    assert np.allclose(f, plain, rtol=1e-14) and s == 1.0
    f, s = pdattn.rope_frequencies(dims, base, pdattn.ROPE_LINEAR, 4.0)
    assert np.allclose(f, plain / 4, rtol=1e-14) and s == 1.0
    f, s = pdattn.rope_frequencies(dims, base, pdattn.ROPE_BASE, 4.0)
    assert s == 1.0 and f[0] == 1.0
    if dims > 2:   # the slowest pair turns `factor` times slower, whatever the number of pairs
        assert np.isclose(f[-1], plain[-1] / 4, rtol=1e-12) and np.all(np.diff(f) < 0)


@pytest.mark.parametrize("dims", [64, 96, 128])
def test_yarn_and_wavelength(dims):
    base, factor, trained = 10000.0, 8.0, 4096.0
    plain, _ = pdattn.rope_frequencies(dims, base)
    turns = trained * plain / (2 * np.pi)
    f, s = pdattn.rope_frequencies(dims, base, pdattn.ROPE_YARN, factor, trained)
    assert np.isclose(s, 0.1 * np.log(8.0) + 1, rtol=1e-7)
    lo = np.floor(dims * np.log(trained / (32 * 2 * np.pi)) / (2 * np.log(base)))
    hi = np.ceil(dims * np.log(trained / (1 * 2 * np.pi)) / (2 * np.log(base)))
    ramp = np.interp(np.arange(dims // 2), [lo, hi], [0.0, 1.0])
    assert np.allclose(f, plain * (1 - ramp) + plain / factor * ramp, rtol=1e-12)
    assert np.all(f[turns > 40] == plain[turns > 40]) and np.allclose(f[turns < 0.7], plain[turns < 0.7] / factor)
    f, s = pdattn.rope_frequencies(dims, base, pdattn.ROPE_WAVELENGTH, factor, trained, 1.0, 4.0)
    assert s == 1.0
    keep = np.interp(turns, [1.0, 4.0], [0.0, 1.0])
    assert np.allclose(f, plain * keep + plain / factor * (1 - keep), rtol=1e-12)


@pytest.mark.parametrize("args", [(0,), (3,), (130,), (-2,), (64, 1.0), (64, float("nan")), (64, 1e4, 5), (64, 1e4, -1),
                                  (64, 1e4, 1, 0.5), (64, 1e4, 1, float("inf")), (64, 1e4, 3, 2.0, 0.0),
                                  (64, 1e4, 3, 2.0, 4096.0, 0.0), (64, 1e4, 4, 2.0, 4096.0, 4.0, 4.0),
                                  (64, 1e4, 4, 2.0, 4096.0, 4.0, 1.0), (64, 1e4, 4, 2.0, float("nan"))])
def test_frequency_refusals(args):
    with pytest.raises(pdattn.PdattnError) as e:
        pdattn.rope_frequencies(*args)
    assert e.value.status == 1


# ---- CPU: the restatement ---------------------------------------------------------------------------

def _turned(x, positions, freq, rotary, interleaved, scale):
    """By complex numbers."""
    y = x.astype(np.float64).copy()
    turn = scale * np.exp(1j * np.outer(positions, freq))[:, None, :]
    r = y[..., :rotary]
    u, w = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rotary // 2], r[..., rotary // 2:])
    z = (u + 1j * w) * turn
    y[..., :rotary] = np.stack([z.real, z.imag], -1).reshape(r.shape) if interleaved else np.concatenate([z.real, z.imag], -1)
    return y


def _restated(fault="none"):
    rng = np.random.default_rng(0)
    good = True
    for rotary, inter in ((128, False), (128, True), (64, False), (20, True), (2, False)):
        x = rng.standard_normal((5, 3, 128)).astype(np.float16)
        pos, freq = rng.integers(0, 10 ** 6, 5), pdattn.rope_frequencies(rotary)[0]
        good &= np.allclose(oracle.rope(x, pos, freq, rotary, inter, 1.3, fault),
                            _turned(x, pos, freq, rotary, inter, 1.3), atol=1e-8)
    return good


def test_restatement_is_complex_multiplication():
    assert _restated()


@pytest.mark.parametrize("fault", [f for f in oracle.ROPE_FAULTS if f != "none"])
def test_planted_fault_is_caught(fault):
    assert not _restated(fault)


# ---- CPU: refusals ------------------------------------------------------------------------------------

def _fake(**kw):
    p = pdattn.RopeAppendParams()
    for name, _ in p._fields_[:12]:
        setattr(p, name, 1 << 20)
    p.n, p.B, p.Hq, p.Hkv, p.rotary_dim, p.scale = 4, 2, 8, 2, 64, 1.0
    p.q_stride, p.k_stride, p.v_stride = 8 * 128, 2 * 128, 2 * 128
    p.q_out = 1 << 24
    for name, x in kw.items():
        setattr(p, name, x)
    return p


@pytest.mark.parametrize("kw", [dict(n=-1), dict(B=-1), dict(Hkv=0), dict(Hq=-1), dict(rotary_dim=0), dict(rotary_dim=63),
                                dict(rotary_dim=130), dict(scale=float("nan")), dict(q=None), dict(Hq=0), dict(k_new=None),
                                dict(v_new=None), dict(q_out=None), dict(k_cache=None), dict(v_cache=None), dict(kv_indptr=None),
                                dict(kv_indices=None), dict(batch_idx=None), dict(positions=None), dict(freq=None),
                                dict(q=(1 << 20) + 8), dict(k_new=(1 << 20) + 2), dict(v_cache=(1 << 20) + 4), dict(q_stride=1023),
                                dict(q_stride=1020), dict(k_stride=250), dict(v_stride=128), dict(q_out=1 << 20, q_stride=1040)])
def test_refusals(kw):
    with pytest.raises(pdattn.PdattnError) as e:
        pdattn.rope_append_kv(_fake(**kw))
    assert e.value.status == 1


@pytest.mark.parametrize("kw", [dict(q=(1 << 24) + 2048), dict(q=(1 << 24) - 16), dict(k_new=(1 << 24) + 8176), dict(v_new=(1 << 24) - 512),
                                dict(q_stride=1 << 22), dict(q=1 << 24, v_new=(1 << 24) + 4096)])
def test_outputs_over_inputs_are_refused(kw):
    with pytest.raises(pdattn.PdattnError) as e:
        pdattn.rope_append_kv(_fake(**kw))
    assert e.value.status == 1 and "overlaps" in str(e.value)


def test_no_tokens():
    pdattn.rope_append_kv(_fake(n=0))
    pdattn.rope_append_kv(_fake(n=0, q=None, k_new=None, v_new=None, q_out=None))   # as empty tensors give


# ---- GPU ----------------------------------------------------------------------------------------------

def _case(lens, Hq, Hkv, bidx, pos, rotary, interleaved=False, scaling="plain", far=0, seed=1, fused=False, inplace=False, no_q=False):
    import torch
    from _gpu import DeviceBatch, device
    bt = inputs.make_batch(lens, max(Hq, Hkv), Hkv, seed)
    db, dev, n = DeviceBatch(bt), device(), len(bidx)
    rng = np.random.default_rng(seed)
    rows = rng.standard_normal((n, Hq + 2 * Hkv, 128)).astype(np.float16)
    both = torch.from_numpy(rows).to(dev)
    q, kn, vn = both[:, :Hq], both[:, Hq:Hq + Hkv], both[:, Hq + Hkv:]
    if not fused:
        q, kn, vn = q.contiguous(), kn.contiguous(), vn.contiguous()
    freq, scale = pdattn.rope_frequencies(rotary, 10000.0, SCALINGS[scaling], 1.0 if scaling == "plain" else 8.0, 4096.0)
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(dev)  # noqa: E731
    bi, po = put(bidx), put(pos)
    rp = put(np.asarray(pos) + far) if far else None
    q_out = q if inplace else torch.full((n, Hq, 128), float("nan"), dtype=torch.float16, device=dev)
    bad = torch.zeros(1, dtype=torch.int32, device=dev)
    f = torch.from_numpy(freq).to(dev)
    tag = f"rope Hq={Hq} Hkv={Hkv} n={n} rotary={rotary} inter={interleaved} {scaling} far={far} fused={fused} inplace={inplace}"
    print(tag, flush=True)
    p = pdattn.make_rope_append_params(None if no_q else q, kn, vn, q_out, db.k, db.v, db.indptr, db.indices, bi, po, f, bt.B,
                                       rotary_dim=rotary, interleaved=interleaved, scale=scale, rope_positions=rp, n_invalid=bad)
    pdattn.rope_append_kv(p)
    torch.cuda.synchronize()
    where = np.asarray(pos, np.int64) + far
    exact = oracle.rope(rows[:, :Hq + Hkv], where, freq, rotary, interleaved, scale)
    half, x = rotary // 2, np.abs(rows[:, :Hq + Hkv, :rotary].astype(np.float64))
    tol = np.zeros(exact.shape)
    if interleaved:
        both = np.repeat(x[..., 0::2] + x[..., 1::2], 2, -1)
    else:
        both = np.concatenate([x[..., :half] + x[..., half:]] * 2, -1)
    tol[..., :rotary] = 2 ** -20 * scale * both + np.maximum(2 ** -11 * np.abs(exact[..., :rotary]), 2 ** -25)
    if not no_q:
        err = np.abs(q_out.float().cpu().numpy() - exact[:, :Hq])
        assert np.all(err <= tol[:, :Hq]), (tag, err.max())
    # k: the rows that the library wrote, at the places where the restatement of the append puts marks
    mark_k = np.repeat(np.arange(1, n + 1, dtype=np.uint16), Hkv * 128).reshape(n, Hkv, 128).view(np.float16)
    kc, vc, nbad = oracle.append_kv(np.zeros_like(bt.k), bt.v, mark_k, rows[:, Hq + Hkv:], bidx, pos, bt.indptr, bt.indices)
    assert int(bad.item()) == nbad
    assert np.array_equal(db.v.cpu().numpy().view(np.uint16), vc.view(np.uint16))
    got, token = db.k.cpu().numpy(), kc.view(np.uint16).astype(np.int64) - 1
    written = token[..., 0, 0] >= 0
    assert np.array_equal(got[~written].view(np.uint16), bt.k[~written].view(np.uint16))
    t = token[..., 0, 0][written]
    err = np.abs(got[written].astype(np.float64) - exact[t, Hq:])
    assert np.all(err <= tol[t, Hq:]), (tag, err.max())
    # the dims that are not rotated come as they were
    assert np.array_equal(got[written][..., rotary:].view(np.uint16), rows[t, Hq:Hq + Hkv][..., rotary:].view(np.uint16))


LENS = [37, 16, 1, 300]


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [128, 64, 32, 16, 96, 2, 6, 20, 126, 48])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_sizes(rotary, interleaved):
    _case(LENS, 8, 2, np.arange(4), np.array(LENS) - 1, rotary, interleaved, seed=rotary)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv", [(32, 8), (64, 8), (32, 32), (16, 2), (3, 3), (7, 1), (1, 1)])
@pytest.mark.parametrize("scaling", ["plain", "yarn", "base"])
def test_heads(Hq, Hkv, scaling):
    _case(LENS, Hq, Hkv, np.arange(4), np.array(LENS) - 1, 128, False, scaling, seed=5)


@pytest.mark.gpu
@pytest.mark.parametrize("far", [10 ** 4, 10 ** 6, 2 ** 31 - 400])
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(far, interleaved):
    _case(LENS, 8, 2, np.arange(4), np.array(LENS) - 1, 128, interleaved, far=far, seed=7)


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [128, 20])
@pytest.mark.parametrize("interleaved", [False, True])
def test_slices_of_one_tensor_and_in_place(rotary, interleaved):
    _case(LENS, 8, 2, np.arange(4), np.array(LENS) - 1, rotary, interleaved, seed=9, fused=True)
    _case(LENS, 8, 2, np.arange(4), np.array(LENS) - 1, rotary, interleaved, seed=9, inplace=True)


@pytest.mark.gpu
def test_keys_alone():
    _case(LENS, 0, 2, np.arange(4), np.array(LENS) - 1, 64, seed=11, no_q=True)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,lens", [(8, 2, [500, 1500, 37]), (4, 1, [3000, 300]), (2, 2, [4000]), (32, 8, [700, 650])])
@pytest.mark.parametrize("rotary,interleaved", [(128, False), (36, False), (64, True)])
def test_prefill_shuffled_with_invalid_tokens(Hq, Hkv, lens, rotary, interleaved):
    """Every position of every sequence in random order, padding tokens (no sequence) and positions past the pages among
    them: q of every token is rotated, whatever becomes of its k and v."""
    rng = np.random.default_rng(Hkv)
    bidx = np.concatenate([np.full(L, b) for b, L in enumerate(lens)])
    pos = np.concatenate([np.arange(L) for L in lens])
    bad_b = rng.choice([-1, len(lens), 0], size=41)
    bad_p = np.where(bad_b == 0, -(-lens[0] // 16) * 16 + rng.integers(0, 100, 41), -rng.integers(0, 9, 41))
    bidx, pos = np.concatenate([bidx, bad_b]), np.concatenate([pos, bad_p])
    order = rng.permutation(len(bidx))
    _case(lens, Hq, Hkv, bidx[order], pos[order], rotary, interleaved, seed=13)


@pytest.mark.gpu
def test_positions_at_the_ends_of_32_bits():
    """No page holds them: nothing is written but q."""
    _case([20], 4, 2, np.zeros(3, int), np.array([2 ** 31 - 1, -2 ** 31, -1]), 128, seed=15)
