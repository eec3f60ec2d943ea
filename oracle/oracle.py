"""ctypes binding of the fp64 CPU oracle (oracle/pdattn_oracle.c).

TEST INFRASTRUCTURE ONLY: imported by tests/, by ``__graft_entry__.smoke()`` as the checker and
by the CPU-baseline leg of ``bench.py``. The product library never loads it.

Each wrapper names the reference function it restates (qilem/cuda-kernel-lab,
01_decode_attention.cu); the C file carries the same citations.
"""
from __future__ import annotations

import ctypes
import os
import subprocess

import numpy as np

HEAD_DIM = 128
PAGE = 16

_HERE = os.path.dirname(os.path.abspath(__file__))
_LIB_PATH = os.path.join(_HERE, "_build", "liboracle.so")
_lib = None

FAULTS = {
    "none": 0,
    "page_off_by_one": 1,
    "kvh_modulo": 2,
    "no_scale": 3,
    "full_last_page": 4,
    "lse_no_max": 5,
    "slot_transpose": 6,
    "merge_no_weight": 7,
    "half_trunc": 8,
    "prefix_no_private": 9,
}


def build(force: bool = False) -> str:
    """Compile the oracle with gcc (oracle/Makefile) and return the library path."""
    if force or not os.path.exists(_LIB_PATH):
        subprocess.run(["make", "-C", _HERE] + (["-B"] if force else []), check=True,
                       stdout=subprocess.DEVNULL)
    return _LIB_PATH


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(_LIB_PATH):
            build()
        L = ctypes.CDLL(_LIB_PATH)
        P = ctypes.c_void_p
        i, d = ctypes.c_int, ctypes.c_double
        L.oracle_half_to_double.argtypes = [ctypes.c_uint16]
        L.oracle_half_to_double.restype = d
        L.oracle_double_to_half.argtypes = [d]
        L.oracle_double_to_half.restype = ctypes.c_uint16
        L.oracle_decode_mt.argtypes = [P] * 6 + [i, i, i, i, d, P, P, i]
        L.oracle_decode_mt.restype = None
        L.oracle_partials.argtypes = [P] * 6 + [i] * 8 + [d, P, P]
        L.oracle_partials.restype = None
        L.oracle_merge.argtypes = [P, P, i, i, P, P]
        L.oracle_merge.restype = None
        L.oracle_shared_prefix_pages.argtypes = [P, P, i]
        L.oracle_shared_prefix_pages.restype = i
        L.oracle_plan_chunks_ref.argtypes = [i, i, i, i, i, ctypes.POINTER(i), ctypes.POINTER(i)]
        L.oracle_plan_chunks_ref.restype = None
        L.oracle_set_fault.argtypes = [i]
        L.oracle_set_fault.restype = None
        _lib = L
    return _lib


class fault:
    """Context manager that plants one named mistake in the oracle (test use only)."""

    def __init__(self, name: str):
        self.code = FAULTS[name]

    def __enter__(self):
        lib().oracle_set_fault(self.code)
        return self

    def __exit__(self, *exc):
        lib().oracle_set_fault(0)
        return False


def _ptr(a: np.ndarray):
    return a.ctypes.data_as(ctypes.c_void_p)


def _u16(a) -> np.ndarray:
    a = np.asarray(a)
    if a.dtype == np.float16:
        a = a.view(np.uint16)
    return np.ascontiguousarray(a, dtype=np.uint16)


def _i32(a) -> np.ndarray:
    return np.ascontiguousarray(np.asarray(a), dtype=np.int32)


def half_to_double(bits: int) -> float:
    return lib().oracle_half_to_double(int(bits))


def double_to_half(x: float) -> int:
    return lib().oracle_double_to_half(float(x))


def decode(q, k, v, indptr, indices, last, Hq: int, Hkv: int, kv_start: int = 0,
           sm_scale: float | None = None, threads: int = 1):
    """fp64 decode attention over the paged cache (01_decode_attention.cu:370-400).

    Returns (out [B, Hq, 128] float64, lse [B, Hq] float64)."""
    q, k, v = _u16(q), _u16(k), _u16(v)
    indptr, indices, last = _i32(indptr), _i32(indices), _i32(last)
    B = len(indptr) - 1
    if sm_scale is None:
        sm_scale = 1.0 / np.sqrt(HEAD_DIM)
    if indices.size == 0:
        indices = np.zeros(1, np.int32)
    out = np.zeros((B, Hq, HEAD_DIM), np.float64)
    lse = np.zeros((B, Hq), np.float64)
    lib().oracle_decode_mt(_ptr(q), _ptr(k), _ptr(v), _ptr(indptr), _ptr(indices), _ptr(last),
                           B, Hq, Hkv, kv_start, float(sm_scale), _ptr(out), _ptr(lse), int(threads))
    return out, lse


def partials(q, k, v, indptr, indices, last, Hq: int, Hkv: int, num_chunks: int,
             chunk_tokens: int, kv_start: int = 0, sm_scale: float | None = None):
    """Per-chunk normalized partial states with uniform chunks (01_decode_attention.cu:88-97,
    228-235). Returns (part_o [B*Hq, num_chunks, 128], part_lse [B*Hq, num_chunks])."""
    q, k, v = _u16(q), _u16(k), _u16(v)
    indptr, indices, last = _i32(indptr), _i32(indices), _i32(last)
    B = len(indptr) - 1
    if sm_scale is None:
        sm_scale = 1.0 / np.sqrt(HEAD_DIM)
    if indices.size == 0:
        indices = np.zeros(1, np.int32)
    po = np.zeros((B * Hq, num_chunks, HEAD_DIM), np.float64)
    pl = np.zeros((B * Hq, num_chunks), np.float64)
    lib().oracle_partials(_ptr(q), _ptr(k), _ptr(v), _ptr(indptr), _ptr(indices), _ptr(last),
                          B, Hq, Hkv, num_chunks, chunk_tokens, kv_start, 0, num_chunks,
                          float(sm_scale), _ptr(po), _ptr(pl))
    return po, pl


def merge(part_o, part_lse):
    """Log-sum-exp merge over the chunk axis (01_decode_attention.cu:238-255).

    part_o [rows, C, 128], part_lse [rows, C] -> (out [rows, 128], lse [rows])."""
    po = np.ascontiguousarray(part_o, dtype=np.float64)
    pl = np.ascontiguousarray(part_lse, dtype=np.float64)
    rows, C = pl.shape
    out = np.zeros((rows, HEAD_DIM), np.float64)
    lse = np.zeros(rows, np.float64)
    lib().oracle_merge(_ptr(po), _ptr(pl), rows, C, _ptr(out), _ptr(lse))
    return out, lse


def shared_prefix_pages(indptr, indices) -> int:
    """Longest shared run of leading physical pages, one private page kept
    (01_decode_attention.cu:634-646)."""
    indptr, indices = _i32(indptr), _i32(indices)
    if indices.size == 0:
        indices = np.zeros(1, np.int32)
    return int(lib().oracle_shared_prefix_pages(_ptr(indptr), _ptr(indices), len(indptr) - 1))


def plan_chunks_ref(resident_blocks: int, B: int, Hkv: int, max_len: int, force_chunks: int = 0):
    """The reference's uniform chunk rule (01_decode_attention.cu:289-312)."""
    nc, ct = ctypes.c_int(), ctypes.c_int()
    lib().oracle_plan_chunks_ref(resident_blocks, B, Hkv, max_len, force_chunks,
                                 ctypes.byref(nc), ctypes.byref(ct))
    return nc.value, ct.value


APPEND_FAULTS = ("none", "slot_kvh_transpose", "page_off_by_one", "position_minus_one")


def append_kv(k_cache, v_cache, k_new, v_new, batch_idx, positions, indptr, indices,
              fault: str = "none"):
    """Paged KV append, restated on the host: token t, at position p of sequence b, is written to
    page indices[indptr[b] + p // 16], slot p % 16, for every kv head -- the page addressing of
    01_decode_attention.cu:112 used for writes (FlashInfer's append convention: the page table
    already covers the appended tokens). Tokens whose sequence or position is out of range are
    skipped and counted. Caches are [num_pages, 16, Hkv, 128] (any 2-byte dtype), new rows
    [n, Hkv, 128]. `fault` plants a mistake for the tests that pin this function.

    Returns (k_cache', v_cache', n_invalid)."""
    kc, vc = np.array(k_cache, copy=True), np.array(v_cache, copy=True)
    indptr, indices = np.asarray(indptr), np.asarray(indices)
    B = len(indptr) - 1
    bad = 0
    for t in range(len(batch_idx)):
        b, p = int(batch_idx[t]), int(positions[t])
        if fault == "position_minus_one":
            p -= 1
        if b < 0 or b >= B or p < 0 or p >= (indptr[b + 1] - indptr[b]) * PAGE:
            bad += 1
            continue
        j = indptr[b] + p // PAGE + (1 if fault == "page_off_by_one" else 0)
        j = min(j, len(indices) - 1)
        page, slot = int(indices[j]), p % PAGE
        if fault == "slot_kvh_transpose":
            # rows laid out [kvh][slot] instead of [slot][kvh]
            flat_k, flat_v = kc[page].reshape(-1, HEAD_DIM), vc[page].reshape(-1, HEAD_DIM)
            Hkv = kc.shape[2]
            for h in range(Hkv):
                flat_k[(h * PAGE + slot) % (PAGE * Hkv)] = k_new[t, h]
                flat_v[(h * PAGE + slot) % (PAGE * Hkv)] = v_new[t, h]
            continue
        kc[page, slot] = k_new[t]
        vc[page, slot] = v_new[t]
    return kc, vc, bad



# ---- drafted tokens -----------------------------------------------------------------------------

TREE_FAULTS = ("none", "mask_transposed", "chain_excludes_self", "context_shifted", "bias_before_cap", "bias_sign",
               "window_inclusive", "sink_in_window_only", "slot_positions", "group_modulo")


def _sequence(indptr, indices, last, b):
    """Page ids and length of sequence b (a last-page length outside [1, 16] is clamped)."""
    pages = np.asarray(indices)[int(indptr[b]):int(indptr[b + 1])]
    return pages, (len(pages) - 1) * PAGE + min(PAGE, max(1, int(last[b]))) if len(pages) else 0


def tree_attention(q, k, v, indptr, indices, last, Hq: int, Hkv: int, q_indptr=None, mask=None, depth=None,
                   sm_scale=None, soft_cap: float = 0.0, slopes=None, window: int = 0, sink: int = 0,
                   max_tokens: int = 512, fault: str = "none"):
    """Attention of drafted tokens in 64 bits, from the definition: token i of sequence b, cached at ctx + i
    (ctx = length - tokens), sees every key below ctx and key ctx + j if bit j of its mask row is set (j <= i
    without a mask); scores sm_scale q.k, capped by cap tanh(x / cap), plus slope (key position - query
    position), positions being ctx + depth (the index without depths, a negative one 0); with a window only keys
    less than it before the query, or below `sink`. Keys not seen are not read.

    Returns (out [n, Hq, 128], lse [n, Hq], slack) where slack holds what a 32-bit evaluation's error is
    proportional to: "weight" [n, Hq, 128] = sum p |v|; "score" [n, Hq] = sum p e and "score_v" [n, Hq, 128] =
    sum p e |v|, e being a score's error bound in units of 2^-24: 136 sum_d |q_d k_d| sm_scale (the products'
    sum) + 16 (|x| + |bias|) (what follows it); "keys" [n, Hq] the keys seen. Tokens of no sequence: NaN.
    `fault` plants a mistake for the tests that pin this function."""
    q = np.asarray(q).astype(np.float64)
    n_tokens = q.shape[0]
    B, G = len(indptr) - 1, Hq // Hkv
    q_indptr = np.arange(B + 1) if q_indptr is None else np.asarray(q_indptr)
    sm = 1.0 / np.sqrt(HEAD_DIM) if sm_scale is None else sm_scale
    out, lse = np.full((n_tokens, Hq, HEAD_DIM), np.nan), np.full((n_tokens, Hq), np.nan)
    slack = {"weight": np.zeros_like(out), "score": np.zeros_like(lse), "score_v": np.zeros_like(out),
             "keys": np.zeros_like(lse)}
    for b in range(B):
        pages, length = _sequence(indptr, indices, last, b)
        q0, n = int(q_indptr[b]), int(q_indptr[b + 1]) - int(q_indptr[b])
        ctx = length - n + (1 if fault == "context_shifted" else 0)
        flat = np.repeat(np.asarray(pages, np.int64) * PAGE, PAGE) + np.tile(np.arange(PAGE), len(pages))
        flat = flat[:length]
        dep = np.arange(n) if depth is None or fault == "slot_positions" else np.maximum(0, np.asarray(depth)[q0:q0 + n])
        j = np.arange(length) - ctx
        drafted = j >= 0
        # position of every key relative to ctx
        pos_k = np.where(drafted, dep[np.clip(j, 0, max(n - 1, 0))] if n else 0, j)
        look = []   # per token: which keys it sees, and how far before it they are
        for i in range(n):
            if mask is None:
                seen = ~drafted | (j <= i - (1 if fault == "chain_excludes_self" else 0))
            else:
                m = np.asarray(mask).view(np.uint32)
                jj = np.clip(j, 0, 32 * m.shape[1] - 1)
                bits = m[q0 + i, jj // 32] >> (jj % 32) & 1
                if fault == "mask_transposed":
                    jj = np.clip(jj, 0, n - 1)
                    bits = m[q0 + jj, i // 32] >> np.uint32(i % 32) & 1
                seen = ~drafted | ((bits != 0) & (j < 32 * m.shape[1]))
            if mask is not None or depth is not None:
                seen &= j < max_tokens
            apart = dep[i] - pos_k
            if window > 0:
                near = apart < window + (1 if fault == "window_inclusive" else 0)
                seen &= near if fault == "sink_in_window_only" else near | (np.arange(length) < sink)
            look.append((i, apart, np.flatnonzero(seen)))
        for kvh in range(Hkv):
            heads = [h for h in range(Hq) if (h % Hkv if fault == "group_modulo" else h // G) == kvh]
            kb = np.asarray(k).reshape(-1, Hkv, HEAD_DIM)[flat, kvh].astype(np.float64)
            vb = np.asarray(v).reshape(-1, Hkv, HEAD_DIM)[flat, kvh].astype(np.float64)
            for i, apart, at in look:
                t = q0 + i
                if len(at) == 0:
                    out[t, heads], lse[t, heads] = 0.0, -np.inf
                    continue
                kk, vv = (kb, vb) if len(at) == length else (kb[at], vb[at])
                for h in heads:
                    x = kk @ q[t, h] * sm
                    e = 136 * (np.abs(kk) @ np.abs(q[t, h])) * abs(sm)
                    bias = np.zeros(len(at)) if slopes is None else float(slopes[h]) * -apart[at]
                    if fault == "bias_sign":
                        bias = -bias
                    if fault == "bias_before_cap":
                        x = x + bias
                    if soft_cap > 0:
                        x = soft_cap * np.tanh(x / soft_cap)
                    if fault != "bias_before_cap":
                        x = x + bias
                    e = e + 16 * (np.abs(x) + np.abs(bias))
                    top = x.max()
                    w = np.exp(x - top)
                    p = w / w.sum()
                    out[t, h], lse[t, h] = p @ vv, top + np.log(w.sum())
                    slack["weight"][t, h] = p @ np.abs(vv)
                    slack["score"][t, h], slack["score_v"][t, h] = p @ e, (p * e) @ np.abs(vv)
                    slack["keys"][t, h] = len(at)
    return out, lse, slack


ROPE_FAULTS = ("none", "other_pairing", "sign", "half_of_head", "scale_twice")


def rope(x, positions, freq, rotary_dim: int, interleaved: bool = False, scale: float = 1.0, fault: str = "none"):
    """Rotary positions in 64 bits: pair (u, w) of the first rotary_dim dims of x [n, heads, 128], at angle
    a = position * freq, becomes scale (u cos a - w sin a, w cos a + u sin a)."""
    x = np.asarray(x).astype(np.float64)
    y = x.copy()
    if fault == "other_pairing":
        interleaved = not interleaved
    if fault == "half_of_head":
        rotary_dim = min(HEAD_DIM, 2 * rotary_dim)
        freq = np.resize(freq, rotary_dim // 2)
    for t, p in enumerate(np.asarray(positions)):
        for i in range(rotary_dim // 2):
            u, w = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)
            a = float(p) * float(freq[i]) * (-1 if fault == "sign" else 1)
            s = scale * scale if fault == "scale_twice" else scale
            y[t, :, u] = s * (x[t, :, u] * np.cos(a) - x[t, :, w] * np.sin(a))
            y[t, :, w] = s * (x[t, :, w] * np.cos(a) + x[t, :, u] * np.sin(a))
    return y


ACCEPT_FAULTS = ("none", "from_the_front", "keys_only", "descending")


def accept_kv(k_cache, v_cache, indptr, indices, last, q_indptr, accepted_indptr, accepted, fault: str = "none"):
    """The rows of the accepted drafted tokens to the front of each sequence's drafted range: list entry i of
    sequence b moves position ctx + accepted[i] to ctx + i. A list that does not ascend within the sequence's
    tokens is counted and its sequence left alone. Returns (k_cache', v_cache', n_invalid)."""
    kc, vc = np.array(k_cache, copy=True), np.array(v_cache, copy=True)
    bad = 0
    for b in range(len(indptr) - 1):
        lst = np.asarray(accepted)[int(accepted_indptr[b]):int(accepted_indptr[b + 1])].astype(np.int64)
        if len(lst) == 0:
            continue
        pages, length = _sequence(indptr, indices, last, b)
        n = int(q_indptr[b + 1]) - int(q_indptr[b])
        ctx = length - n
        if n < 0 or ctx < 0 or lst.min() < 0 or lst.max() >= n or np.any(np.diff(lst) <= 0):
            bad += 1
            continue
        base = 0 if fault == "from_the_front" else ctx
        order = range(len(lst) - 1, -1, -1) if fault == "descending" else range(len(lst))
        for i in order:
            src, dst = ctx + lst[i], base + i
            s, d = (pages[src // PAGE], src % PAGE), (pages[dst // PAGE], dst % PAGE)
            kc[d] = kc[s]
            if fault != "keys_only":
                vc[d] = vc[s]
    return kc, vc, bad
