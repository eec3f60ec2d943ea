"""The operators of a speculative decoding step next to the decode attention: what a serving loop has them do on one GPU.

A case is one pass on data that is already on the GPU, of one of
    rope     the rotary positions of new tokens' q and k, and the paged append of k and v
    tree     the attention of drafted tokens (a tree with an ancestor mask, or a chain) over the paged cache
    scored   the same attention for one token per sequence, with capped scores, a distance bias or a window
    accept   the accepted drafted tokens' rows moved to the front of the drafted range of the cache
q, K and V are fp16 N(0, 1), pages are scattered over the cache at random, head_dim is 128 and a page holds 16
tokens. The lengths of a ragged batch are part of the case (``lens_seed``), its values come from the seed.

    own                     False: run() is the operators' plain form; True: the library's kernels
    listed()                the cases
    draw(rng)               one more case of the same ranges
    prepare(case, seed)     inputs on the GPU
    run(state)              one pass; returns its outputs
    work(case)              bytes and operations the pass cannot do without
    exact(case, seed)       the outputs in 64 bits
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DIM = 128
PAGE = 16

# The most K and V bytes, operations and scores (of the padded batch) of a drawn attention, and bytes of a drawn append.
MOST_KV_BYTES = 270e6
MOST_FLOPS = 130e9
MOST_SCORES = 3e8
MOST_ROPE_BYTES = 8e8

# (Hq, Hkv): MHA, and groups of 2, 4 and 8 query heads per kv head.
HEADS = [(32, 8), (32, 8), (64, 8), (64, 8), (32, 32), (16, 16), (16, 8), (16, 4), (64, 16), (16, 2)]


def listed():
    return [
        # a decode step: one new token of each of 64 sequences, whole head rotated, halves paired
        _case("rope_decode64", "rope", 32, 8, 64, 256, 4096, n=(1, 1), rotary=128, lens_seed=3),
        # drafted tokens far beyond the trained context, frequencies scaled by YaRN's ramp, eight heads per kv head
        _case("rope_draft_far", "rope", 64, 8, 16, 512, 2048, n=(33, 33), rotary=128, scaling="yarn", far=900_000,
              lens_seed=5),
        # prefill: long prompts, half of each head rotated, neighbouring pairs, q, k and v in one projection's output
        _case("rope_prefill32k", "rope", 32, 8, 8, 4096, 4096, n=(4096, 4096), rotary=64, interleaved=True,
              scaling="linear", fused=True, lens_seed=7),
        # one user, a small tree of drafted tokens: the smallest verification, where launches and latency count
        _case("tree_1x2k_n16", "tree", 32, 8, 1, 2048, 2048, n=(16, 16), tree=True, lens_seed=11),
        # a serving batch of long contexts, 64 drafted tokens each: many rows on every key
        _case("tree_8x8k_n64", "tree", 32, 8, 8, 8192, 8192, n=(64, 64), tree=True, lens_seed=13),
        # ragged contexts and trees, eight query heads per kv head
        _case("tree_ragged32_g8", "tree", 64, 8, 32, 200, 6000, n=(5, 27), tree=True, lens_seed=17),
        # a chunk of a prefill over a cached context: 512 new tokens in order, no mask in memory
        _case("chain_2x8k_n512", "tree", 32, 8, 2, 8192, 8192, n=(512, 512), lens_seed=19),
        # decode with capped scores, ragged contexts
        _case("capped_ragged32", "scored", 32, 8, 32, 200, 6000, cap=50.0, lens_seed=23),
        # one long context with a distance bias, one query head per kv head
        _case("bias_1x32k_mha", "scored", 16, 16, 1, 32768, 32768, bias=True, lens_seed=29),
        # a window with the first keys kept, capped scores, contexts longer than the window
        _case("window1k_64", "scored", 64, 8, 64, 1024, 8192, cap=30.0, window=1024, sink=4, lens_seed=31),
        # the end of a verification: the accepted path of each of 64 sequences
        _case("accept_64", "accept", 32, 8, 64, 40, 400, n=(64, 64), lens_seed=37),
        # one user, a short path
        _case("accept_1", "accept", 32, 8, 1, 300, 300, n=(16, 16), lens_seed=41),
    ]


def _case(name, kind, Hq, Hkv, B, lo, hi, n=(1, 1), tree=False, cap=0.0, bias=False, window=0, sink=0, rotary=0,
          interleaved=False, scaling="none", far=0, fused=False, lens_seed=1):
    """B sequences with lo .. hi cached tokens before the n[0] .. n[1] new ones each; tree: the new tokens form a tree
    (else a chain); rotary: dims rotated, far: added to the rotary positions, fused: q, k and v are slices of one
    tensor."""
    return {"name": name, "kind": kind, "Hq": Hq, "Hkv": Hkv, "B": B, "lo": lo, "hi": hi, "n_lo": n[0], "n_hi": n[1],
            "tree": tree, "cap": cap, "bias": bias, "window": window, "sink": sink, "rotary": rotary,
            "interleaved": interleaved, "scaling": scaling, "far": far, "fused": fused, "lens_seed": lens_seed}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: 1 .. 128 sequences of 1 .. 32768 cached tokens (ragged or equal), 1 .. 512 new ones
    each, every group size, all score parameters, every pairing and scaling, any even number of rotated dims."""
    kind = rng.choice(["rope", "rope", "tree", "tree", "tree", "scored", "scored", "accept"])
    Hq, Hkv = rng.choice(HEADS)
    most = int(MOST_KV_BYTES / (Hkv * DIM * 4))   # tokens whose K and V fit
    B = _log_int(rng, 1, 128)
    more = {"lens_seed": rng.randint(1, 10 ** 6)}
    if kind in ("tree", "scored"):
        hi = _log_int(rng, 16, min(32768, most // B))
        if kind == "tree":
            more["tree"] = rng.random() < 0.7
            top = min(256 if more["tree"] else 512, int(MOST_FLOPS / (4 * DIM * Hq * B * hi)))
            while top > 1 and (B * (hi + top) > most or B * Hq * top * (hi + top) > MOST_SCORES):
                top //= 2
            n_hi = _log_int(rng, 1, max(1, top))
            more["n"] = (n_hi if rng.random() < 0.5 else _log_int(rng, 1, n_hi), n_hi)
        hi = max(1, min(hi, most // B - 1))
        if kind == "scored" or rng.random() < 0.4:
            more["cap"] = rng.choice([0.0, 15.0, 30.0, 50.0])
            more["bias"] = rng.random() < 0.4
            if rng.random() < 0.4:
                more["window"] = _log_int(rng, 16, max(17, hi))
                more["sink"] = rng.choice([0, 0, 4, 20])
    elif kind == "rope":
        hi = _log_int(rng, 1, 4096)
        top = max(1, min(4096, int(MOST_ROPE_BYTES / (4 * DIM * (Hq + 2 * Hkv))) // B, most // 2 // B))
        n_hi = 1 if rng.random() < 0.3 else _log_int(rng, 1, top)
        more["n"] = (n_hi if rng.random() < 0.5 else _log_int(rng, 1, n_hi), n_hi)
        hi = max(1, min(hi, most // 2 // B))
        more["rotary"] = rng.choice([128, 128, 64, 32, 96, 2 * rng.randint(1, 64)])
        more["interleaved"] = rng.random() < 0.5
        more["scaling"] = rng.choice(["none", "linear", "base", "yarn", "wavelength"])
        more["far"] = rng.choice([0, 0, _log_int(rng, 1000, 10 ** 6)])
        more["fused"] = rng.random() < 0.5
    else:
        hi = _log_int(rng, 1, 1024)
        n_hi = _log_int(rng, 2, 256)
        more["n"] = (n_hi if rng.random() < 0.5 else _log_int(rng, 1, n_hi), n_hi)
    lo = hi if rng.random() < 0.3 else _log_int(rng, max(1, hi // 32), hi)
    c = _case("", kind, Hq, Hkv, B, lo, hi, **more)
    del c["name"]
    return c


def _sizes(case):
    """(cached tokens before the new ones, new tokens) of every sequence."""
    rng = np.random.default_rng(case["lens_seed"])

    def spread(lo, hi):
        return np.exp(rng.uniform(math.log(lo), math.log(hi), case["B"])).round().astype(np.int64).clip(lo, hi)

    return spread(case["lo"], case["hi"]), spread(case["n_lo"], case["n_hi"])


def _frequencies(case):
    """Radians per position of each pair of rotated dims, and the factor of cos and sin: contexts of 4096 scaled to
    eight times as many. none: base ** (-2 i / dims); linear: divided by 8; base: of base * 8 ** (dims / (dims - 2));
    yarn and wavelength: slow dims divided, fast ones kept, a ramp between (over the dims, over the wavelengths)."""
    dims, base, factor, trained = case["rotary"], 10000.0, 8.0, 4096.0
    i = np.arange(dims // 2, dtype=np.float64)
    f, scale = base ** (-2 * i / dims), 1.0
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "base" and dims > 2:
        f = (base * factor ** (dims / (dims - 2))) ** (-2 * i / dims)
    elif case["scaling"] == "yarn":
        lo, hi = (dims * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), dims - 1)
        keep = 1 - ((i - lo) / max(hi - lo, 1e-3)).clip(0, 1)
        f, scale = f / factor * (1 - keep) + f * keep, 0.1 * math.log(factor) + 1
    elif case["scaling"] == "wavelength":
        turns = trained * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clip(0, 1)
        f = f / factor * (1 - keep) + f * keep
    return f, scale


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    rng = np.random.default_rng(int(seed))
    ctx, new = _sizes(case)
    B, Hq, Hkv, lens = case["B"], case["Hq"], case["Hkv"], ctx + new

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float16)

    def ints(x):
        return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(dev)

    pages = -(-lens // PAGE)
    indptr = np.concatenate([[0], np.cumsum(pages)])
    starts = np.concatenate([[0], np.cumsum(new)])
    total = int(starts[-1])
    seqs = np.repeat(np.arange(B), new)
    index = np.arange(total) - starts[seqs]
    s = dict(case, total=total, max_len=int(lens.max()), max_new=int(new.max()), device=dev,
             k=normal(int(indptr[-1]), PAGE, Hkv, DIM), v=normal(int(indptr[-1]), PAGE, Hkv, DIM), indptr=ints(indptr),
             indices=ints(rng.permutation(int(indptr[-1]))), last=ints(lens - (pages - 1) * PAGE), starts=ints(starts),
             stream=torch.cuda.current_stream())
    if case["kind"] == "accept":
        # a path from a tree: each token a few further on than the one before, as many as are accepted
        take = np.minimum(new, rng.integers(1, 10, B))
        s["accepted"] = ints(np.concatenate([np.sort(rng.choice(new[b], take[b], replace=False)) for b in range(B)]))
        s["accepted_starts"] = ints(np.concatenate([[0], np.cumsum(take)]))
        return s
    if case["kind"] == "rope":
        if case["fused"]:
            qkv = normal(total, (Hq + 2 * Hkv), DIM)
            s["q"], s["k_new"], s["v_new"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        else:
            s["q"], s["k_new"], s["v_new"] = normal(total, Hq, DIM), normal(total, Hkv, DIM), normal(total, Hkv, DIM)
        f, s["scale"] = _frequencies(case)
        s["freq"] = torch.from_numpy(f).to(dev)
        s["seqs"], s["pos"] = ints(seqs), ints(ctx[seqs] + index)
        s["rope_pos"] = ints(ctx[seqs] + index + case["far"])
        s["q_out"] = torch.empty(total, Hq, DIM, dtype=torch.float16, device=dev)
        return s
    s["q"] = normal(total, Hq, DIM)
    s["out"] = torch.empty(total, Hq, DIM, dtype=torch.float16, device=dev)
    s["lse"] = torch.empty(total, Hq, dtype=torch.float32, device=dev)
    s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device=dev) if case["bias"] else None
    s["mask"] = s["depth"] = None
    if case["kind"] == "tree" and case["tree"]:
        # every token's parent is one of the tokens before it, or none; the ancestors by doubling of the paths
        n = s["max_new"]
        parent = torch.rand(B, n, generator=g, device=dev) * torch.arange(1, n + 1, device=dev) - 1
        parent = parent.ceil().long().clamp_(min=-1)
        reach = torch.zeros(B, n, n + 1, device=dev).scatter_(2, (parent % (n + 1)).unsqueeze(2), 1.0)[:, :, :n]
        reach = reach + torch.eye(n, device=dev)
        for _ in range(max(1, (n - 1).bit_length())):
            reach = (torch.bmm(reach, reach) > 0).float()
        words = -(-n // 32)
        bits = torch.nn.functional.pad(reach, (0, 32 * words - n)).view(B, n, words, 32).double()
        bits = (bits * 2.0 ** torch.arange(32, device=dev, dtype=torch.float64)).sum(3).long()
        at = torch.from_numpy(seqs).to(dev), torch.from_numpy(index).to(dev)
        s["mask"] = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).int()[at].contiguous()
        s["depth"] = (reach.sum(2) - 1).int()[at].contiguous()
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"rope": _rope, "accept": _accept}.get(s["kind"], _attend)(s)


# ---- the library's kernels ------------------------------------------------------------------------------------------

_kept = {}


def _library():
    """The binding, and one workspace for the process, which grows to what the calls need."""
    if not _kept:
        path = os.path.abspath("cuda-kernel-lab_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import pdattn
        _kept["pdattn"], _kept["ws"] = pdattn, pdattn.Workspace()
    return _kept["pdattn"], _kept["ws"]


def _run_own(s):
    pdattn, ws = _library()
    kind = s["kind"]
    if kind == "accept":
        pdattn.accept_kv(s["k"], s["v"], s["indptr"], s["indices"], s["last"], s["starts"], s["accepted_starts"],
                         s["accepted"], s["B"], s["Hkv"], stream=s["stream"])
        return s["k"], s["v"]
    if kind == "rope":
        if "params" not in s:   # the argument block, built once for its buffers
            s["params"] = pdattn.make_rope_append_params(
                s["q"], s["k_new"], s["v_new"], s["q_out"], s["k"], s["v"], s["indptr"], s["indices"], s["seqs"],
                s["pos"], s["freq"], s["B"], rotary_dim=s["rotary"], interleaved=s["interleaved"], scale=s["scale"],
                rope_positions=s["rope_pos"])
        pdattn.rope_append_kv(s["params"], stream=s["stream"])
        return s["q_out"], s["k"], s["v"]
    if "params" not in s:
        tree = kind == "tree"
        s["params"] = pdattn.make_tree_params(
            s["q"], s["k"], s["v"], s["indptr"], s["indices"], s["last"], s["B"], s["Hq"], s["Hkv"],
            q_indptr=s["starts"] if tree else None, max_tokens=s["max_new"], mask=s["mask"], depth=s["depth"],
            soft_cap=s["cap"], slopes=s["slopes"], window=s["window"], sink=s["sink"])
    pdattn.tree_attention(s["params"], s["out"], s["lse"], ws, stream=s["stream"])
    return s["out"], s["lse"]


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _rotated(x, s):
    """The rows of x [tokens, heads, 128] rotated by their positions: angles in 64 bits, the rotation in 32."""
    a = s["rope_pos"].double()[:, None] * s["freq"]
    cos, sin = (a.cos() * s["scale"]).float()[:, None], (a.sin() * s["scale"]).float()[:, None]
    x = x.float()
    r, half = s["rotary"], s["rotary"] // 2
    if s["interleaved"]:
        u, w = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([u * cos - w * sin, w * cos + u * sin], -1).flatten(-2)
    else:
        u, w = x[..., :half], x[..., half:r]
        y = torch.cat([u * cos - w * sin, w * cos + u * sin], -1)
    return torch.cat([y, x[..., r:]], -1).half()


def _rope(s):
    pos = s["pos"].long()
    page = s["indices"][s["indptr"][s["seqs"].long()].long() + pos // PAGE].long()
    s["k"][page, pos % PAGE] = _rotated(s["k_new"], s)
    s["v"][page, pos % PAGE] = s["v_new"]
    return _rotated(s["q"], s), s["k"], s["v"]


def _accept(s):
    a = s["accepted_starts"].long()
    count = a[1:] - a[:-1]
    seq = torch.repeat_interleave(torch.arange(s["B"], device=s["device"]), count, output_size=s["accepted"].numel())
    pages, indptr, starts = s["indices"], s["indptr"].long(), s["starts"].long()
    length = (indptr[1:] - indptr[:-1] - 1) * PAGE + s["last"]
    first = (length - (starts[1:] - starts[:-1]))[seq]
    to = first + torch.arange(seq.numel(), device=s["device"]) - a[seq]
    src = first + s["accepted"]
    at_src, at_to = ((pages[indptr[seq] + p // PAGE].long(), p % PAGE) for p in (src, to))
    s["k"][at_to], s["v"][at_to] = s["k"][at_src], s["v"][at_src]
    return s["k"], s["v"]


def _attend(s):
    B, Hq, Hkv, dev = s["B"], s["Hq"], s["Hkv"], s["device"]
    G, n, most = Hq // Hkv, s["max_new"], -(-s["max_len"] // PAGE)
    indptr, starts = s["indptr"].long(), s["starts"].long()
    length = ((indptr[1:] - indptr[:-1] - 1) * PAGE + s["last"])[:, None]
    count = (starts[1:] - starts[:-1])[:, None]
    first = length - count
    # the sequences' keys and values, padded to the longest
    entry = (indptr[:-1, None] + torch.arange(most, device=dev)).clamp_(max=s["indices"].numel() - 1)
    page = s["indices"][entry].long()
    k = s["k"][page].view(B, most * PAGE, Hkv, DIM).permute(0, 2, 3, 1).float().contiguous()
    v = s["v"][page].view(B, most * PAGE, Hkv, DIM).permute(0, 2, 1, 3).float().contiguous()
    # the queries, padded to the most: rows (token, head of the group)
    token = (starts[:-1, None] + torch.arange(n, device=dev)).clamp_(max=s["total"] - 1)
    q = s["q"][token].view(B, n, Hkv, G, DIM).permute(0, 2, 1, 3, 4).reshape(B, Hkv, n * G, DIM).float()
    x = torch.matmul(q, k) * (1.0 / math.sqrt(DIM))
    if s["cap"] > 0:
        x = torch.tanh(x / s["cap"]) * s["cap"]
    x = x.view(B, Hkv, n, G, most * PAGE)
    at = torch.arange(most * PAGE, device=dev)
    draft = at - first                                      # [B, keys]: index among the new tokens, or below 0
    valid = (at < length)[:, None]                          # [B, 1, keys]
    own_index = torch.arange(n, device=dev)
    if s["mask"] is None:
        seen = draft[:, None] <= own_index[:, None]
        depth, depth_key = own_index.expand(B, n), draft
    else:
        j = draft.clamp(0, n - 1)
        words = s["mask"][token].long()                     # [B, n, words]
        word = torch.gather(words, 2, (j // 32)[:, None].expand(B, n, -1))
        seen = ((word >> (j % 32)[:, None]) & 1).bool() | (draft < 0)[:, None]
        depth = s["depth"][token].long()
        depth_key = torch.where(draft >= 0, torch.gather(depth, 1, j), draft)
    apart = (first + depth)[:, :, None] - (first + depth_key)[:, None]   # [B, n, keys]: query's position - key's
    if s["window"] > 0:
        seen = seen & ((apart < s["window"]) | (at < s["sink"]))
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, Hkv, 1, G, 1) * apart[:, None, :, None].float()
    x = x.masked_fill(~(seen & valid)[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(x - top)
    norm = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, n * G, -1), v).view(B, Hkv, n, G, DIM) / norm.clamp(min=1e-30)
    lse = (top + torch.log(norm)).squeeze(-1)
    # back to one row per token
    real = own_index < count
    out = o.permute(0, 2, 1, 3, 4).reshape(B, n, Hq, DIM)[real].half()
    return out, lse.permute(0, 2, 1, 3).reshape(B, n, Hq)[real]


# ---- bytes and operations, and 64 bits ------------------------------------------------------------------------------

def work(case):
    ctx, new = _sizes(case)
    Hq, Hkv, total = case["Hq"], case["Hkv"], int(new.sum())
    row = 2 * DIM
    table = 4 * int((2 + -(-(ctx + new) // PAGE)).sum())
    if case["kind"] == "rope":
        return {"bytes": total * (2 * row * (Hq + 2 * Hkv) + 12) + 4 * case["rotary"], "flops": 3 * case["rotary"] * total * (Hq + Hkv)}
    if case["kind"] == "accept":
        take = np.minimum(new, 5)   # 1 .. 9 of them are accepted, and most of those move
        return {"bytes": int(take.sum()) * (2 * 2 * row * Hkv + 8), "flops": 0}
    keys = ctx + new
    if case["window"]:
        keys = np.minimum(keys, np.minimum(ctx, case["window"] + case["sink"]) + new)
    visible = keys - new + 1   # of each new token, at least
    mask = 4 * int((new * -(-new // 32)).sum()) if case["tree"] else 0
    return {"bytes": 2 * row * Hkv * int(keys.sum()) + total * Hq * (2 * row + 4) + table + mask,
            "flops": 4 * DIM * Hq * int((new * visible).sum())}


def exact(case, seed):
    s = prepare(case, seed)
    ctx, new = _sizes(case)
    indptr, starts, Hkv = s["indptr"].cpu().numpy(), s["starts"].cpu().numpy(), case["Hkv"]
    G, table = case["Hq"] // Hkv, s["indices"].long()

    def place(b, positions):
        positions = torch.as_tensor(positions, device=s["device"])
        return table[int(indptr[b]) + positions // PAGE], positions % PAGE

    if case["kind"] == "accept":
        path, at = s["accepted"].cpu().numpy(), s["accepted_starts"].cpu().numpy()
        for cache in (s["k"], s["v"]):
            for b in range(case["B"]):
                for i, a in enumerate(path[at[b]:at[b + 1]].tolist()):   # in order: a row is read before it is written
                    cache[place(b, [int(ctx[b]) + i])] = cache[place(b, [int(ctx[b]) + a])]
        return s["k"], s["v"]
    if case["kind"] == "rope":
        angle = torch.outer(s["rope_pos"].double(), s["freq"])
        turn = torch.polar(torch.full_like(angle, s["scale"]), angle)[:, None]

        def rotated(x):
            x, r = x.double(), case["rotary"]
            pairs = x[..., :r].unflatten(-1, (r // 2, 2)) if case["interleaved"] else x[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
            y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            y = y.flatten(-2) if case["interleaved"] else y.transpose(-1, -2).flatten(-2)
            return torch.cat([y, x[..., r:]], -1)

        k, v, k_new = s["k"].double(), s["v"].double(), rotated(s["k_new"])
        for b in range(case["B"]):
            rows = slice(int(starts[b]), int(starts[b + 1]))
            at = place(b, s["pos"][rows].long())
            k[at], v[at] = k_new[rows], s["v_new"][rows].double()
        return rotated(s["q"]), k, v
    out = torch.zeros(s["total"], case["Hq"], DIM, dtype=torch.float64, device=s["device"])
    lse = torch.full((s["total"], case["Hq"]), -math.inf, dtype=torch.float64, device=s["device"])
    for b in range(case["B"]):
        c, m = int(ctx[b]), int(new[b])
        rows, keys = slice(int(starts[b]), int(starts[b + 1])), torch.arange(c + m, device=s["device"])
        depth = torch.arange(m, device=s["device"]) if s["depth"] is None else s["depth"][rows].long()
        sees = torch.ones(m, c + m, dtype=torch.bool, device=s["device"])
        if s["mask"] is None:
            sees[:, c:] = torch.ones(m, m, dtype=torch.bool, device=s["device"]).tril()
        else:
            j = torch.arange(m, device=s["device"])
            sees[:, c:] = (s["mask"][rows].long()[:, j // 32] >> (j % 32)) & 1 != 0
        apart = (c + depth)[:, None] - torch.cat([keys[:c], c + depth])
        if case["window"]:
            sees &= (apart < case["window"]) | (keys < case["sink"])
        page, slot = place(b, keys)
        for h in range(case["Hq"]):   # one query head at a time: [tokens, 128] in 64 bits
            kh, vh = s["k"][page, slot, h // G].double(), s["v"][page, slot, h // G].double()
            x = s["q"][rows, h].double() @ kh.T / math.sqrt(DIM)
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["bias"]:
                x = x - s["slopes"][h].double() * apart
            x = x.masked_fill(~sees, -math.inf)
            lse[rows, h] = torch.logsumexp(x, 1)
            out[rows, h] = torch.softmax(x, 1) @ vh
    return out, lse
