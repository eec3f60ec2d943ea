"""The drafted-token operators as torch ops (pdattn.torch_ops): registered, with the shapes that a tracer needs, refusals; on the
GPU a step of them against the direct calls bit for bit, on a stream of the caller's and traced."""
import numpy as np
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import pdattn
import pdattn.torch_ops  # noqa: F401  (registers torch.ops.pdattn.*)
from _draft import check_attention, make_draft, oracle_attention

SCALE = float(1.0 / np.sqrt(128.0))


def _tensors(dr, dev):
    t = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    i = lambda x: t(np.asarray(x, np.int32))  # noqa: E731
    bt = dr.bt
    return dict(q=t(dr.q), k_cache=t(bt.k), v_cache=t(bt.v), kv_indptr=i(bt.indptr), kv_indices=i(bt.indices),
                kv_last_page_len=i(bt.last), sm_scale=SCALE, q_indptr=i(dr.q_indptr), max_tokens=dr.max_tokens, mask=i(dr.mask),
                depth=i(dr.depth))


def _rope_args(x, n, Hq, Hkv, dev):
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(n, Hq + 2 * Hkv, 128, generator=g).half().to(dev)
    freq, scale = pdattn.rope_frequencies(64, 10000.0)
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    return (qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], x["k_cache"], x["v_cache"], x["kv_indptr"], x["kv_indices"],
            i([0, 0, 1]), i([3, 4, 2]), torch.from_numpy(freq).to(dev), True, scale)


def test_fake_shapes():
    dr = make_draft([40, 7], [5, 3], 8, 2, seed=1)
    x = _tensors(dr, "cpu")
    with FakeTensorMode() as mode:
        f = {k: mode.from_tensor(v) if isinstance(v, torch.Tensor) else v for k, v in x.items()}
        out, lse = torch.ops.pdattn.tree_attention(**f, window=20)
        assert out.shape == (8, 8, 128) and out.dtype == torch.float16 and lse.shape == (8, 8) and lse.dtype == torch.float32
        args = [mode.from_tensor(v) if isinstance(v, torch.Tensor) else v for v in _rope_args(x, 3, 8, 2, "cpu")]
        assert torch.ops.pdattn.rope_append_kv(*args).shape == (3, 8, 128)
        acc = [mode.from_tensor(torch.zeros(n, dtype=torch.int32)) for n in (3, 1)]
        assert torch.ops.pdattn.accept_kv(f["k_cache"], f["v_cache"], f["kv_indptr"], f["kv_indices"], f["kv_last_page_len"],
                                          f["q_indptr"], *acc) is None


@pytest.mark.parametrize("change,error", [
    (dict(q=lambda q: q.float()), TypeError), (dict(q=lambda q: q[..., :64]), ValueError), (dict(q_indptr=lambda x: x.long()), TypeError),
    (dict(q_indptr=lambda x: x[:-1].contiguous()), ValueError), (dict(mask=lambda x: x[:-1].contiguous()), ValueError),
    (dict(kv_indptr=lambda x: x[:-1].contiguous()), ValueError), (dict(depth=lambda x: x[1:].contiguous()), ValueError),
    (dict(k_cache=lambda x: x[:, :8]), ValueError), (dict(v_cache=lambda x: x[:-1]), ValueError),
    (dict(k_cache=lambda x: x.bfloat16()), TypeError), (dict(slopes=lambda _: torch.zeros(3)), ValueError),
    (dict(q_indptr=lambda _: None), ValueError), (dict(kv_indices=lambda x: torch.stack([x, x], 1)[:, 0]), TypeError),
])
def test_refusals(change, error):
    x = _tensors(make_draft([40, 7], [5, 3], 8, 2, seed=1), "cpu")
    for k, f in change.items():
        x[k] = f(x.get(k))
    with pytest.raises(error):
        torch.ops.pdattn.tree_attention(**x)


@pytest.mark.gpu
@pytest.mark.parametrize("score", [dict(), dict(soft_cap=10.0, window=90, sink=2)])
def test_attention_is_the_library_s(score):
    from _draft import DeviceDraft
    dr = make_draft([300, 17, 64], [7, 40, 1], 16, 2, seed=5)
    print("op: tree_attention", flush=True)
    out, lse = torch.ops.pdattn.tree_attention(**_tensors(dr, "cuda:0"), **score)
    torch.cuda.synchronize()
    direct = DeviceDraft(dr).run(**score)
    assert np.array_equal(out.float().cpu().numpy(), direct[0]) and np.array_equal(lse.cpu().numpy(), direct[1])
    check_attention(*direct, oracle_attention(dr, **score), "op")


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_are_defined():
    dr = make_draft([30, 17], [3, 4], 8, 2, seed=7, extra_rows=5)
    out, lse = torch.ops.pdattn.tree_attention(**_tensors(dr, "cuda:0"))
    assert (out[7:] == 0).all() and torch.isneginf(lse[7:]).all() and torch.isfinite(lse[:7]).all()


@pytest.mark.gpu
def test_a_traced_step_on_a_side_stream():
    """Rotate and append, attend, accept, as one traced graph, against the direct calls on copies."""
    dev = torch.device("cuda:0")
    dr = make_draft([40, 7], [5, 3], 8, 2, seed=9)
    x = _tensors(dr, dev)
    direct = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in x.items()}
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    acc = (i([0, 2, 3]), i([1, 4, 2]))

    def step(x, rope):
        q = torch.ops.pdattn.rope_append_kv(*rope)
        y = dict(x, q=torch.cat([q, x["q"][3:]]))
        out, lse = torch.ops.pdattn.tree_attention(**y)
        torch.ops.pdattn.accept_kv(x["k_cache"], x["v_cache"], x["kv_indptr"], x["kv_indices"], x["kv_last_page_len"], x["q_indptr"], *acc)
        return out, lse

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        print("op: traced step", flush=True)
        out, lse = torch.compile(step, backend="aot_eager", fullgraph=True)(x, _rope_args(x, 3, 8, 2, dev))
    side.synchronize()
    rope = _rope_args(direct, 3, 8, 2, dev)
    q = torch.empty(3, 8, 128, dtype=torch.float16, device=dev)
    pdattn.rope_append_kv(pdattn.make_rope_append_params(*rope[:3], q, *rope[3:10], 2, rotary_dim=64, interleaved=True, scale=rope[11]))
    direct["q"] = torch.cat([q, direct["q"][3:]])
    d_out, d_lse = torch.empty_like(direct["q"]), torch.empty(8, 8, device=dev)
    ws, d = pdattn.Workspace(), direct
    pdattn.tree_attention(pdattn.make_tree_params(d["q"], d["k_cache"], d["v_cache"], d["kv_indptr"], d["kv_indices"],
                                                  d["kv_last_page_len"], 2, 8, 2, q_indptr=d["q_indptr"], max_tokens=d["max_tokens"],
                                                  mask=d["mask"], depth=d["depth"], sm_scale=SCALE), d_out, d_lse, ws)
    pdattn.accept_kv(d["k_cache"], d["v_cache"], d["kv_indptr"], d["kv_indices"], d["kv_last_page_len"], d["q_indptr"], *acc, 2, 2)
    torch.cuda.synchronize()
    pdattn.workspace_release(ws)
    assert torch.equal(out, d_out) and torch.equal(lse, d_lse)
    assert torch.equal(x["k_cache"], d["k_cache"]) and torch.equal(x["v_cache"], d["v_cache"])


@pytest.mark.gpu
def test_nothing_to_do():
    """No tokens, no sequences, no pages, nothing accepted."""
    dev = "cuda:0"
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    h = lambda *shape: torch.ones(shape, dtype=torch.float16, device=dev)  # noqa: E731
    ops, kc, vc = torch.ops.pdattn, h(2, 16, 2, 128), h(2, 16, 2, 128)
    out, lse = ops.tree_attention(h(0, 8, 128), kc, vc, i(0), i(), i(), SCALE, q_indptr=i(0))
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)
    out, lse = ops.tree_attention(h(3, 8, 128), kc, vc, i(0, 0), i(), i(0), SCALE, q_indptr=i(0, 3), max_tokens=3)
    assert (out == 0).all() and torch.isneginf(lse).all()
    freq = torch.from_numpy(pdattn.rope_frequencies(64)[0]).to(dev)
    assert ops.rope_append_kv(h(0, 8, 128), h(0, 2, 128), h(0, 2, 128), kc, vc, i(0, 1), i(1), i(), i(), freq).shape == (0, 8, 128)
    ops.accept_kv(kc, vc, i(0, 1), i(1), i(3), i(0, 2), i(0, 0), i())
    assert (kc == 1).all() and (vc == 1).all()
