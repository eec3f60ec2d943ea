// append.hip -- the write side of the paged caches: the append of new tokens' K/V (the step before decode),
// the same with the rotary positions of q and k, and the move of accepted drafted tokens' rows.
//
// Layout of the caches and the page table as in the decode path (qilem/cuda-kernel-lab,
// 01_decode_attention.cu:5-9, 112; FlashInfer's page-table convention): element (page, slot,
// kvh, d) at ((page*16 + slot)*Hkv + kvh)*128 + d. The page table already describes the caches
// after the append (the caller allocates pages and sets kv_indptr / kv_last_page_len first, as
// with FlashInfer's append_paged_kv_cache); token t, at position pos[t] of sequence b[t], goes to
// page kv_indices[kv_indptr[b] + pos / 16], slot pos % 16.
//
// Byte work, HBM-bound. A workgroup of 256 threads takes several tokens, 4096 16-byte pieces of
// K and V in all (16 tokens at Hkv = 8, 16 pieces per thread). One thread per token resolves the
// token's page slot from the page table into LDS; meanwhile every thread has already issued the
// loads of its pieces, which do not depend on the page table, so the table's dependent loads
// overlap the data loads, and after one barrier the pieces are stored. A token's Hkv rows are
// contiguous both in the input [n, Hkv, 128] and in its page slot ([16, Hkv, 128] per page), so
// reads and writes are coalesced runs. A token whose position lies outside its sequence's pages
// is not written; it is counted in *n_invalid.
#include <algorithm>

#include "pdattn_internal.h"

namespace pdattn {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kAppendThreads = 256;
constexpr int kAppendPieces = 16;                                  // 16-byte pieces per thread per pass
constexpr int kAppendMaxTokens = kAppendThreads * kAppendPieces / 32;   // at Hkv = 1

// the most tokens a workgroup takes: as many as fill one pass of kAppendPieces pieces per thread
inline int append_max_tokens_per_wg(int Hkv) {
    const int ppt = 2 * Hkv * (kHeadDim / 8);
    return ppt >= kAppendThreads * kAppendPieces ? 1 : kAppendThreads * kAppendPieces / ppt;
}

__global__ __launch_bounds__(kAppendThreads) void append_kv_kernel(AppendArgs a) {
    __shared__ long long s_dst[kAppendMaxTokens];   // first piece of the token's slot row, or -1
    const int tid = threadIdx.x;
    const int row_pieces = a.Hkv * (kHeadDim / 8);  // 16-byte pieces of one token's K (or V)
    const int ppt = 2 * row_pieces;                 // per token: K then V
    const int tpb = a.tpb;
    const size_t t0 = (size_t)blockIdx.x * tpb;
    const int ntok = (int)min((size_t)tpb, (size_t)a.n - t0);

    if (tpb == 1) {   // one token (a decode step's few tokens): its slot is uniform, no LDS hand-off
        const int b = a.batch_idx[t0], pos = a.positions[t0];
        const bool ok_b = b >= 0 && b < a.B;
        const int pb = ok_b ? a.kv_indptr[b] : 0, np = ok_b ? a.kv_indptr[b + 1] - pb : 0;
        if (!ok_b || pos < 0 || pos >= np * kPage) {
            if (tid == 0 && a.n_invalid) atomicAdd(a.n_invalid, 1);
            return;
        }
        const size_t page = (size_t)(uint32_t)a.kv_indices[pb + pos / kPage];
        const size_t dst = (page * kPage + pos % kPage) * row_pieces;
        const u32x4* kn = reinterpret_cast<const u32x4*>(a.k_new) + t0 * row_pieces;
        const u32x4* vn = reinterpret_cast<const u32x4*>(a.v_new) + t0 * row_pieces;
        u32x4* kc = reinterpret_cast<u32x4*>(a.k_cache) + dst;
        u32x4* vc = reinterpret_cast<u32x4*>(a.v_cache) + dst;
        for (int pc = tid; pc < ppt; pc += kAppendThreads) {
            if (pc < row_pieces) kc[pc] = kn[pc];
            else vc[pc - row_pieces] = vn[pc - row_pieces];
        }
        return;
    }

    if (tid < ntok) {
        const size_t t = t0 + tid;
        const int b = a.batch_idx[t], pos = a.positions[t];
        const bool ok_b = b >= 0 && b < a.B;
        const int pb = ok_b ? a.kv_indptr[b] : 0, np = ok_b ? a.kv_indptr[b + 1] - pb : 0;
        long long dst = -1;
        if (ok_b && pos >= 0 && pos < np * kPage) {
            const size_t page = (size_t)(uint32_t)a.kv_indices[pb + pos / kPage];
            dst = (long long)((page * kPage + pos % kPage) * row_pieces);
        } else if (a.n_invalid && blockIdx.y == 0) {
            atomicAdd(a.n_invalid, 1);
        }
        s_dst[tid] = dst;
    }

    const u32x4* kn = reinterpret_cast<const u32x4*>(a.k_new) + t0 * row_pieces;
    const u32x4* vn = reinterpret_cast<const u32x4*>(a.v_new) + t0 * row_pieces;
    u32x4* kc = reinterpret_cast<u32x4*>(a.k_cache);
    u32x4* vc = reinterpret_cast<u32x4*>(a.v_cache);
    const int total = ntok * ppt;
    for (int base = 0; base < tpb * ppt; base += kAppendThreads * kAppendPieces) {   // uniform
        u32x4 val[kAppendPieces];
#pragma unroll
        for (int u = 0; u < kAppendPieces; ++u) {
            const int idx = base + u * kAppendThreads + tid;
            if (idx < total) {
                const int tok = idx / ppt, pc = idx % ppt;
                val[u] = pc < row_pieces ? kn[(size_t)tok * row_pieces + pc]
                                         : vn[(size_t)tok * row_pieces + pc - row_pieces];
            }
        }
        __syncthreads();   // the slots in s_dst
#pragma unroll
        for (int u = 0; u < kAppendPieces; ++u) {
            const int idx = base + u * kAppendThreads + tid;
            if (idx < total) {
                const int tok = idx / ppt, pc = idx % ppt;
                const long long dst = s_dst[tok];
                if (dst >= 0) {
                    if (pc < row_pieces) kc[dst + pc] = val[u];
                    else vc[dst + pc - row_pieces] = val[u];
                }
            }
        }
    }
}

// ---- rotary positions and the append in one pass -------------------------------------------------
//
// A token's rows (its Hq rows of q, Hkv of k, Hkv of v) are moved by 16 lanes each, 16 bytes per lane.
// The pairs of a rotated row are (dim, dim + half), whose other halves lie in another lane of the row's
// 16 (an exchange between lanes), or neighbours, both in the lane. cos and sin of a token's angles are
// worked out once per workgroup, into LDS, while the rows' loads are on the way: the angle p f in 64
// bits, reduced to a fraction of a turn there (p f may be 2^31 radians, of which 32 bits would leave no
// fraction), then sin and cos of pi x in 32 bits. A row is read by one wave before any lane of it writes,
// so q may be rotated in place.
// Byte work, bound by HBM: every row is read once and written once, with non-temporal stores, which do not wait in
// an L2 for the kernel's end: 32768 tokens of 48 rows 154.2 -> 144.3 us (5.6 TB/s; a large copy 5.1), 528 of 80 10.1 -> 8.6, and
// the latter with their attention 67.5 -> 66.6.
constexpr int kRopeThreads = 256;
constexpr int kRopeRows = 4;          // rows of a 16-lane group on the way at once
constexpr int kRopeMaxTokens = 8;     // tokens per workgroup
constexpr int kRopeMaxPairs = kHeadDim / 2;

typedef _Float16 rf16x8 __attribute__((ext_vector_type(8)));

__global__ __launch_bounds__(kRopeThreads) void rope_append_kernel(RopeArgs a) {
    __shared__ float2 s_cs[kRopeMaxTokens][kRopeMaxPairs];
    __shared__ long long s_dst[kRopeMaxTokens];   // byte offset of the token's slot row in the caches, or -1
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15;
    const int R = a.Hq + 2 * a.Hkv, half = a.rotary_dim / 2;
    const int t0 = blockIdx.x * a.tpb, ntok = min(a.tpb, a.n - t0);
    const int row0 = blockIdx.y * a.rows_wg, rows = min(ntok * R, row0 + a.rows_wg);   // the workgroup's: [row0, rows)

    auto source = [&](int row, int& tok, int& r) {
        tok = (int)div_by((uint32_t)row, (uint32_t)R, a.rows_m);
        r = row - tok * R;
        const int64_t t = t0 + tok;
        const char* p = r < a.Hq ? static_cast<const char*>(a.q) + t * a.q_stride + r * 256
                      : r < a.Hq + a.Hkv ? static_cast<const char*>(a.k_new) + t * a.k_stride + (r - a.Hq) * 256
                                         : static_cast<const char*>(a.v_new) + t * a.v_stride + (r - a.Hq - a.Hkv) * 256;
        return p;
    };
    u32x4 val[kRopeRows];
    auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < kRopeRows; ++u) {
            const int row = base + u * (kRopeThreads / 16);
            int tok, r;
            if (row < rows) val[u] = reinterpret_cast<const u32x4*>(source(row, tok, r))[c];
        }
    };
    const int mine = row0 + (tid >> 4);
    load(mine);

    if (tid < ntok && a.Hkv > 0) {
        const int t = t0 + tid, b = a.batch_idx[t], pos = a.positions[t];
        const bool ok_b = b >= 0 && b < a.B;
        const int pb = ok_b ? a.kv_indptr[b] : 0, np = ok_b ? a.kv_indptr[b + 1] - pb : 0;
        long long dst = -1;
        if (ok_b && pos >= 0 && pos / kPage < np) {
            const size_t page = (size_t)(uint32_t)a.kv_indices[pb + pos / kPage];
            dst = (long long)((page * kPage + pos % kPage) * a.Hkv * 256);
        } else if (a.n_invalid && blockIdx.y == 0) {
            atomicAdd(a.n_invalid, 1);
        }
        s_dst[tid] = dst;
    }
    for (int i = tid; i < ntok * half; i += kRopeThreads) {
        const int tok = i / half, pair = i - tok * half, t = t0 + tok;
        const int pos = a.rope_positions ? a.rope_positions[t] : a.positions[t];
        const double turns = (double)pos * a.freq[pair] * 0.15915494309189535;   // 1 / (2 pi)
        float sn, cs;
        sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
        s_cs[tok][pair] = make_float2(cs * a.scale, sn * a.scale);
    }
    __syncthreads();

    for (int base = mine; base - (tid >> 4) < rows; base += kRopeRows * (kRopeThreads / 16)) {   // uniform
        if (base != mine) load(base);
#pragma unroll
        for (int u = 0; u < kRopeRows; ++u) {
            const int row = base + u * (kRopeThreads / 16);
            const bool ok = row < rows;
            int tok = 0, r = 0;
            const char* src = ok ? source(row, tok, r) : nullptr;
            const bool turn = ok && r < a.Hq + a.Hkv && 8 * c < a.rotary_dim;
            rf16x8 x = __builtin_bit_cast(rf16x8, val[u]);
            if (a.interleaved) {
                if (turn) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        if (8 * c + e >= a.rotary_dim) break;
                        const float2 w = s_cs[tok][4 * c + e / 2];
                        const float p = (float)x[e], n = (float)x[e + 1];
                        x[e] = (_Float16)(p * w.x - n * w.y);
                        x[e + 1] = (_Float16)(n * w.x + p * w.y);
                    }
                }
            } else {
                rf16x8 y;
                if (half % 8 == 0) {   // (uniform) the pair's other half is a whole lane's piece
                    const int other = (lane & 48) | ((8 * c < half ? c + half / 8 : c - half / 8) & 15);
                    u32x4 o;
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = (uint32_t)__shfl((int)val[u][i], other, 64);
                    y = __builtin_bit_cast(rf16x8, o);
                } else if (turn) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int d = 8 * c + e, p = d < half ? d + half : d - half;
                        y[e] = d < a.rotary_dim ? reinterpret_cast<const _Float16*>(src)[p] : (_Float16)0.f;
                    }
                }
                if (turn) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int d = 8 * c + e;
                        if (d >= a.rotary_dim) break;
                        const bool lo = d < half;
                        const float2 w = s_cs[tok][lo ? d : d - half];
                        x[e] = (_Float16)((float)x[e] * w.x + (float)y[e] * (lo ? -w.y : w.y));
                    }
                }
            }
            if (!ok) continue;
            const u32x4 res = __builtin_bit_cast(u32x4, x);
            if (r < a.Hq) {
                __builtin_nontemporal_store(res, reinterpret_cast<u32x4*>(static_cast<char*>(a.q_out) + ((int64_t)(t0 + tok) * a.Hq + r) * 256) + c);
            } else if (s_dst[tok] >= 0) {
                const bool is_k = r < a.Hq + a.Hkv;
                char* cache = static_cast<char*>(is_k ? a.k_cache : a.v_cache);
                __builtin_nontemporal_store(res, reinterpret_cast<u32x4*>(cache + s_dst[tok] + (r - a.Hq - (is_k ? 0 : a.Hkv)) * 256) + c);
            }
        }
    }
}

// ---- the accepted drafted tokens' rows ---------------------------------------------------------------
//
// A thread owns one 16-byte column of a sequence's token rows, in K or in V, and moves the list's rows in
// order, kAcceptRows read before the first of them is written. The indices ascend, so index i of the list
// is at least i: a row is written where rows of the list at or before it lay, never one still to be read.
// So no thread waits for another, and the move is in place. Every wave checks the whole list first.
constexpr int kAcceptThreads = 256;
constexpr int kAcceptRows = 8;

__global__ __launch_bounds__(kAcceptThreads) void accept_kv_kernel(AcceptArgs a) {
    const int b = blockIdx.x, lane = threadIdx.x & 63;
    const int row_pieces = a.Hkv * (kHeadDim / 8);
    const int col = blockIdx.y * kAcceptThreads + threadIdx.x;
    const int a0 = a.accepted_indptr[b], m = a.accepted_indptr[b + 1] - a0;
    if (m <= 0) return;
    const int pb = a.kv_indptr[b], np = a.kv_indptr[b + 1] - pb;
    const int len = np > 0 ? (np - 1) * kPage + min(kPage, max(1, a.kv_last[b])) : 0;
    const int n = a.q_indptr[b + 1] - a.q_indptr[b], ctx = len - n;
    bool bad = n < 0 || ctx < 0;
    for (int i = lane; i < m; i += 64) {
        const int x = a.accepted[a0 + i];
        bad |= x < 0 || x >= n || (i > 0 && a.accepted[a0 + i - 1] >= x);
    }
    if (__builtin_amdgcn_ballot_w64(bad)) {
        if (col == 0 && a.n_invalid) atomicAdd(a.n_invalid, 1);
        return;
    }
    if (col >= 2 * row_pieces) return;
    u32x4* cache = reinterpret_cast<u32x4*>(col < row_pieces ? a.k_cache : a.v_cache);
    const int piece = col < row_pieces ? col : col - row_pieces;
    auto place = [&](int index) {
        const int pos = ctx + index;
        const size_t page = (size_t)(uint32_t)a.kv_indices[pb + pos / kPage];
        return (page * kPage + pos % kPage) * row_pieces + piece;
    };
    for (int i0 = 0; i0 < m; i0 += kAcceptRows) {
        u32x4 val[kAcceptRows];
        int from[kAcceptRows];
#pragma unroll
        for (int u = 0; u < kAcceptRows; ++u) from[u] = a.accepted[a0 + min(i0 + u, m - 1)];
#pragma unroll
        for (int u = 0; u < kAcceptRows; ++u) val[u] = cache[place(from[u])];
#pragma unroll
        for (int u = 0; u < kAcceptRows; ++u)
            if (i0 + u < m && from[u] != i0 + u) cache[place(i0 + u)] = val[u];
    }
}

}  // namespace

hipError_t launch_rope_append(const RopeArgs& args, int cus, hipStream_t s) {
    RopeArgs a = args;
    const int rows = a.Hq + 2 * a.Hkv;
    if (a.n <= 0 || rows <= 0) return hipSuccess;
    // one token per workgroup until every CU has some, then enough for kRopeRows rows per lane group
    const int fill = kRopeRows * (kRopeThreads / 16) / rows;
    a.tpb = std::max(1, std::min({kRopeMaxTokens, fill, a.n / std::max(1, 4 * cus)}));
    // few tokens: a token's rows over as many workgroups as the CUs hold at once, a row per lane group at least (64 tokens
    // of 48 rows 5.2 -> 4.2 us; 528 of 80 are the same either way)
    const int parts = a.tpb > 1 ? 1 : std::max(1, std::min(8 * cus / a.n, rows / (kRopeThreads / 16)));
    a.rows_wg = (a.tpb * rows + parts - 1) / parts;
    a.rows_m = div_multiplier((uint32_t)rows);
    rope_append_kernel<<<dim3((a.n + a.tpb - 1) / a.tpb, parts), kRopeThreads, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_accept_kv(const AcceptArgs& a, hipStream_t s) {
    if (a.B <= 0) return hipSuccess;
    const int cols = 2 * a.Hkv * (kHeadDim / 8);
    accept_kv_kernel<<<dim3(a.B, (cols + kAcceptThreads - 1) / kAcceptThreads), kAcceptThreads, 0, s>>>(a);
    return hipGetLastError();
}

// Tokens per workgroup: enough workgroups for every CU first (a decode step's few tokens get one
// each), then up to one full pass per thread (a prefill's many tokens).
hipError_t launch_append_kv(const AppendArgs& args, int cus, hipStream_t s) {
    if (args.n <= 0) return hipSuccess;
    AppendArgs a = args;
    a.tpb = std::max(1, std::min(append_max_tokens_per_wg(a.Hkv), a.n / std::max(1, cus)));
    const size_t grid = ((size_t)a.n + a.tpb - 1) / a.tpb;
    append_kv_kernel<<<(unsigned)grid, kAppendThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace pdattn
