// tree_body.h -- attention of drafted tokens over the paged cache (pdattn_tree_attention): several query
// tokens per sequence, seeing the cached keys before them and, of each other, an ancestor mask's or a
// chain's, with scores that may be capped, biased by distance and windowed. Compiled with cascade.hip.
//
//   x = sm_scale q.k;  x = cap tanh(x / cap);  x += slope_h (pos_k - pos_q);  unseen: -inf
//   out = sum_k softmax(x)_k v_k,  lse = ln sum_k exp(x_k)
//
// The rows of a sequence for one kv head (its tokens times the head's G query heads) are the columns of fp16 MFMAs, as
// in decode_body.h: S^T = K Q^T, O^T += V^T P^T, 16 rows a tile. A workgroup takes up to 16 NT rows; its four waves
// split the keys, each streaming its own 32-key blocks through its own LDS slot by direct loads, with no barrier in
// the loop; at the end of a piece the four states are joined through LDS. Which workgroup does what: tree_arith.h; the
// device finds it from the page table and q_indptr, so that a captured launch serves any lengths.
#pragma once

#include <math.h>

#include "decode_body.h"
#include "tree_arith.h"

namespace pdattn {
namespace {

constexpr float kTreeLn2 = 0.69314718055994531f;
constexpr float kTreeLog2e = 1.4426950408889634f;
constexpr int kTreeMaxTokens = PDATTN_TREE_MAX_TOKENS;
constexpr int kTreeMaskWords = kTreeMaxTokens / 32;
constexpr int kTreeWaves = 4;
constexpr int kTreeThreads = kTreeWaves * 64;
constexpr int kTreeScan = 4;   // sequences per thread of a pass of the scan

// tanh(x) in 32 bits. |x| <= 1: the convergent x (10395 + 1260 z + 21 z^2) / (10395 + 4725 z + 210 z^2 + z^3), z = x^2, of
// x / (1 + x^2 / (3 + x^2 / (5 + ...))) (Lambert), within 5e-10 of it; else 1 - 2 / (e^(2 |x|) + 1), whose 1 no
// longer cancels.
__device__ __forceinline__ float tree_tanh_small(float x) {
    const float z = x * x;
    return x * fmaf(z, fmaf(z, 21.f, 1260.f), 10395.f) *
           __builtin_amdgcn_rcpf(fmaf(z, fmaf(z, z + 210.f, 4725.f), 10395.f));
}
__device__ __forceinline__ float tree_tanh_large(float x) {
    const float e = __builtin_amdgcn_exp2f(2.8853900817779268f * fabsf(x));
    return copysignf(fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f), x);
}

// The kernel's arguments, read again from the kernarg segment where they are used: held in scalar registers
// across a piece they would spill. (Only valid in a kernel's own body, so in force-inlined functions alone.)
typedef const __attribute__((address_space(4))) TreeArgs* TreeArgPtr;
__device__ __forceinline__ TreeArgPtr tree_args() {
    TreeArgPtr p = (TreeArgPtr)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

// ---- the range of a workgroup ---------------------------------------------------------------------

struct TreeScan {
    int64_t wave[2 * kTreeWaves];
    int64_t prefix;   // units before the range's first sequence
    int first;        // that sequence
    int tables[5];    // and its entries, as tree_load_entry
};

template <class A>
__device__ __forceinline__ TreeSeq tree_seq_of(const A& a, int ip0, int ip1, int last, int q0, int q1, int extra) {
    return tree_seq(ip0, ip1, last, q0, q1, a.n_tokens, a.tl, a.window, a.sink, a.mask == nullptr, a.weight, extra);
}

// The entries of two sequences in the device's tables in one register, lanes 0 .. 4 and 8 .. 12: the first page-table
// entries of the sequence and of the next, the tokens in its last page, the first tokens (rows of q) of it and of the next.
// This lane's entry (lane & 7) of sequence b:
template <class A>
__device__ __forceinline__ int tree_load_entry(const A& a, int b, int lane) {
    const int e = lane & 7;
    b = min(b, a.B - 1);
    const int32_t *last = a.kv_last, *ip = a.kv_indptr, *q = a.q_indptr;
    const int32_t* p = e == 2 ? last + b : ip + b + (e == 1);
    if (q && e > 2) p = q + b + (e == 4);
    const int v = *p;
    return e > 2 && !q ? b + (e == 4) : v;
}

__device__ __forceinline__ int64_t tree_shfl_up(int64_t v, int d) {
    const int lo = __shfl_up((int)v, d, 64), hi = __shfl_up((int)(v >> 32), d, 64);
    return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}
__device__ __forceinline__ int64_t tree_uniform(int64_t v) {
    return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int tree_dpp_add(int v) {   // + the value that the DPP step brings, 0 where it brings none
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}

struct TreeFour {   // sequences 4 t .. 4 t + 3 of a pass, t the thread
    int ip[kTreeScan + 1], last[kTreeScan], q[kTreeScan + 1];
    int64_t u[kTreeScan];
};

// The units of the pass's sequences, those before the thread's, and the pass's sum. (All loads at clamped places, so that
// none waits for another.)
template <int NW>
__device__ __forceinline__ int64_t tree_scan_pass(const TreeArgs& a, TreeScan& S, int b0, TreeFour& f, int64_t& sum) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = b0 + kTreeScan * tid;
#pragma unroll
    for (int k = 0; k <= kTreeScan; ++k) f.ip[k] = a.kv_indptr[min(b + k, a.B)];
#pragma unroll
    for (int k = 0; k <= kTreeScan; ++k) f.q[k] = min(b + k, a.B);
    if (a.q_indptr) {
#pragma unroll
        for (int k = 0; k <= kTreeScan; ++k) f.q[k] = a.q_indptr[min(b + k, a.B)];
    }
#pragma unroll
    for (int k = 0; k < kTreeScan; ++k) f.last[k] = a.kv_last[min(b + k, a.B - 1)];
    int64_t mine = 0;
#pragma unroll
    for (int k = 0; k < kTreeScan; ++k) {
        f.u[k] = b + k < a.B ? tree_seq_of(a, f.ip[k], f.ip[k + 1], f.last[k], f.q[k], f.q[k + 1], a.extra).total() : 0;
        mine += f.u[k];
    }
    int64_t x = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t y = tree_shfl_up(x, d);
        if (lane >= d) x += y;
    }
    if (lane == 63) S.wave[wave] = x;
    __syncthreads();
    int64_t before = 0;
    sum = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        before += w < wave ? S.wave[w] : 0;
        sum += S.wave[w];
    }
    __syncthreads();   // (S.wave may be written again)
    return before + x - mine;
}

// Range g of the batch.
struct TreeRange {
    TreeCuts cuts;
    int64_t lo;       // its first unit
    int64_t in;       // that unit within sequence b
    int b, left;      // and the units of the range
    int entries;      // of sequences b and b + 1, as tree_load_entry
    int extra;        // units of an item's start
};
template <int NW>
__device__ __forceinline__ bool tree_find_range(const TreeArgs& a, TreeScan& S, int g, TreeRange& r) {
    const int lane = threadIdx.x & 63;
    if (a.B <= 64) {
        // A sequence per lane, in every wave by itself: no barrier, and 32 bits while no sequence has 2^24 units
        const int b = min(lane, a.B - 1);
        const int32_t *ip = a.kv_indptr, *q = a.q_indptr;
        const int ip0 = ip[b], ip1 = ip[b + 1], last = a.kv_last[b];
        int q0 = b, q1 = b + 1;
        if (q) {
            q0 = q[b];
            q1 = q[b + 1];
        }
        const TreeSeq seq = tree_seq_of(a, ip0, ip1, last, q0, q1, 0);
        int64_t mine = lane < a.B ? seq.total() : 0;
        // Items that are all alike, and a whole number of ranges each: all ranges start one piece, and none has more
        r.extra = a.extra;
        const int u = (int)mine;
        if (a.extra && !__builtin_amdgcn_ballot_w64(lane < a.B && u != __builtin_amdgcn_readfirstlane(u)) &&
            a.ranges % max(1, a.B * __builtin_amdgcn_readfirstlane(seq.groups)) == 0)
            r.extra = 0;
        if (lane < a.B) mine += (int64_t)r.extra * seq.groups;
        if (!__builtin_amdgcn_ballot_w64(mine >> 24 != 0)) {
            int x = (int)mine;   // inclusive sums: within rows of 16 lanes, then from row to row
            x = tree_dpp_add<0x111, 0xF>(x);
            x = tree_dpp_add<0x112, 0xF>(x);
            x = tree_dpp_add<0x114, 0xF>(x);
            x = tree_dpp_add<0x118, 0xF>(x);
            x = tree_dpp_add<0x142, 0xA>(x);
            x = tree_dpp_add<0x143, 0xC>(x);
            r.cuts = tree_cuts(__builtin_amdgcn_readlane(x, 63), a.ranges, a.least_units, a.early, a.late);
            if (g >= r.cuts.ranges) return false;
            r.lo = r.cuts.start(g);
            r.left = (int)(r.cuts.start(g + 1) - r.lo);
            const int before = x - (int)mine, lo = (int)r.lo;
            const uint64_t here = __builtin_amdgcn_ballot_w64(before <= lo && lo < x);
            r.b = here ? __builtin_ctzll(here) : 0;   // (one bit)
            r.in = lo - __builtin_amdgcn_readlane(before, r.b);
            const int n = min(r.b + 1, a.B - 1);
            const int e = lane & 7;
            auto of = [&](int i) {
                const int u0 = __builtin_amdgcn_readlane(ip0, i), u1 = __builtin_amdgcn_readlane(ip1, i), u2 = __builtin_amdgcn_readlane(last, i);
                const int u3 = __builtin_amdgcn_readlane(q0, i), u4 = __builtin_amdgcn_readlane(q1, i);
                return e == 0 ? u0 : e == 1 ? u1 : e == 2 ? u2 : e == 3 ? u3 : u4;
            };
            const int e0 = of(r.b), e1 = of(n);
            r.entries = lane & 8 ? e1 : e0;
            return true;
        }
    }
    r.extra = a.extra;
    constexpr int kPass = kTreeScan * 64 * NW;
    TreeFour f;
    int64_t sum, at = tree_scan_pass<NW>(a, S, 0, f, sum), units = sum;
    for (int b0 = kPass; b0 < a.B; b0 += kPass) {
        (void)tree_scan_pass<NW>(a, S, b0, f, sum);
        units += sum;
    }
    r.cuts = tree_cuts(tree_uniform(units), a.ranges, a.least_units, a.early, a.late);
    if (g >= r.cuts.ranges) return false;
    r.lo = r.cuts.start(g);
    r.left = __builtin_amdgcn_readfirstlane((int)(r.cuts.start(g + 1) - r.lo));
    int64_t before = 0;
    for (int b0 = 0; b0 < a.B; b0 += kPass) {
        if (a.B > kPass) at = tree_scan_pass<NW>(a, S, b0, f, sum);
        int64_t p = before + at;
#pragma unroll
        for (int k = 0; k < kTreeScan; ++k) {
            if (p <= r.lo && r.lo < p + f.u[k]) {
                S.prefix = p;
                S.first = b0 + kTreeScan * (int)threadIdx.x + k;
                S.tables[0] = f.ip[k];
                S.tables[1] = f.ip[k + 1];
                S.tables[2] = f.last[k];
                S.tables[3] = f.q[k];
                S.tables[4] = f.q[k + 1];
            }
            p += f.u[k];
        }
        before += sum;
    }
    __syncthreads();
    r.b = __builtin_amdgcn_readfirstlane(S.first);
    r.in = r.lo - tree_uniform(S.prefix);
    const int after = tree_load_entry(a, r.b + 1, lane);
    r.entries = S.tables[min(lane & 7, 4)];
    r.entries = lane & 8 ? after : r.entries;
    return true;
}

// ---- one piece ------------------------------------------------------------------------------------

// The value itself, as a new value in every call: what is formed from it is not kept across a loop.
__device__ __forceinline__ uint32_t tree_fresh(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}
__device__ __forceinline__ uint32_t tree_fresh_s(uint32_t v) {
    asm volatile("" : "+s"(v));
    return v;
}

// What a piece of any body has in LDS.
template <int NW_, int ROWS_>
struct TreeCommon {
    static constexpr int NW = NW_, THREADS = 64 * NW, ROWS = ROWS_;   // waves
    uint32_t mask[ROWS][kTreeMaskWords];                    // the group's mask rows
    int depth[kTreeMaxTokens];                              // the sequence's drafted tokens' depths
    TreeScan scan;
    int wild[2];                                            // the piece goes row by row (tree_piece_rows)
};
// The key-split body: 16 NT rows, every wave all of them.
template <int NT>
struct TreeSplitShared : TreeCommon<kTreeWaves, 16 * NT> {
    alignas(256) uint8_t slot[kTreeWaves][kDecSlotBytes];   // a block of the wave's; at the end its output
    float m[kTreeWaves][16 * NT];
    float l[kTreeWaves][16 * NT];
    __device__ __forceinline__ uint8_t* scratch(int wave) { return slot[wave]; }
};
static_assert(16 * 2 * kHeadDim * 4 <= kDecSlotBytes, "a wave's output fits its slot");
// The row-split body: 16 NT rows of each of NW waves, and 64-key blocks that all waves read.
constexpr int kTreeBlockBytes = 8 * kDecPageBytes;          // K of four pages, then V of four pages
template <int NW, int NT>
struct TreeWideShared : TreeCommon<NW, 16 * NW * NT> {
    static constexpr int NB = NW == 8 ? 4 : 2;              // blocks
    alignas(256) uint8_t block[NB][kTreeBlockBytes];
    __device__ __forceinline__ uint8_t* scratch(int wave) { return block[0] + 1024 * wave; }
};

struct TreePiece {
    TreeSeq q;
    int pb, q0;            // first page-table entry and first token (row of q) of the sequence
    int i0, tokens, rows;  // the group's first token within the sequence, its tokens and rows
    int p0, p1;            // attended pages of the piece
    int slot;              // partial slot, or -1
    int par;               // which of the flags (TreeCommon) is the piece's
};

// What of a piece is needed again only at its end, or in few blocks, read from the lanes where tree_workgroup keeps it.
struct TreeCold {
    int v;
    __device__ __forceinline__ int i0() const { return __builtin_amdgcn_readlane(v, 20); }
    __device__ __forceinline__ int rows() const { return __builtin_amdgcn_readlane(v, 21); }
    __device__ __forceinline__ int q0() const { return __builtin_amdgcn_readlane(v, 22); }
    __device__ __forceinline__ int slot() const { return __builtin_amdgcn_readlane(v, 23); }
    // the workgroup is of the second half of the grid
    __device__ __forceinline__ int late() const { return __builtin_amdgcn_readlane(v, 24); }
    // (lane 19: the next piece's flag)
    __device__ __forceinline__ int flag() const { return ~__builtin_amdgcn_readlane(v, 19) & 1; }
};

// Not 0 where one of two fp16 is infinite or NaN: exponents of ones carry into the sign's place.
__device__ __forceinline__ uint32_t tree_not_finite(uint32_t w) { return ((w & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }

// (so that sums of positions fit an int)
__device__ __forceinline__ int tree_depth(int d) { return min(max(d, 0), 1 << 28); }

// Position of drafted token j relative to the context, as a key.
template <class Sh>
__device__ __forceinline__ int tree_key_pos(bool depth, const Sh& S, int j) {
    const int d = S.depth[min(max(j, 0), kTreeMaxTokens - 1)];   // (read in any case: without a branch)
    return depth && j >= 0 ? d : j;
}

// Which keys a piece's rows see: none from `end` on (so none in places from p1 on), and every row all keys of the pages at
// places [a0, a1).
struct TreeKeys {
    int end, p1, a0, a1;
};
template <bool MOD, class A>
__device__ __forceinline__ TreeKeys tree_keys(const A& a, const TreePiece& p, int lane) {
    TreeKeys k;
    const TreeSeq& sq = p.q;
    const bool tree = a.mask || a.depth;
    k.end = a.mask ? sq.len : min(sq.len, sq.ctx + p.i0 + p.tokens);
    if (tree) k.end = min(k.end, sq.ctx + kTreeMaxTokens);
    k.p1 = min(p.p1, sq.below(max(0, (k.end + kPage - 1) / kPage)));
    // of the keys below `hi` every row sees those from `lo` on: the window's start at the last position of the group
    const int hi = tree ? sq.ctx : sq.ctx + p.i0 + 1;
    int lo = 0;
    if (MOD && a.window > 0) {
        int last = p.i0 + p.tokens - 1;
        if (a.depth) {
            last = 0;
            for (int i = lane; i < p.tokens; i += 64) last = max(last, tree_depth(a.depth[p.q0 + p.i0 + i]));
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) last = max(last, __shfl_xor(last, d, 64));
            last = __builtin_amdgcn_readfirstlane(last);
        }
        lo = max(0, sq.ctx + last - a.window + 1);
    }
    k.a0 = sq.below((lo + kPage - 1) / kPage);
    k.a1 = sq.below(max(0, hi) / kPage);
    return k;
}

// The mask rows of the group and the depths of the sequence's drafted tokens into LDS, for pieces that hold drafted keys:
// loaded by the first of these, stored by the second, with other loads started in between.
template <class Sh>
struct TreeStage {
    static constexpr int M = Sh::ROWS * kTreeMaskWords / Sh::THREADS, D = kTreeMaxTokens / Sh::THREADS;
    uint32_t m[M];
    int d[D];
};
template <bool MOD, class Sh, class A>
__device__ __forceinline__ void tree_stage_load(TreeStage<Sh>& g, const A& a, const TreePiece& p) {
    const int tid = (int)tree_fresh(threadIdx.x);
    if (a.mask) {
#pragma unroll
        for (int k = 0; k < TreeStage<Sh>::M; ++k) {
            const int r = min((tid + k * Sh::THREADS) / kTreeMaskWords, p.tokens - 1), w = tid % kTreeMaskWords;
            const uint32_t v = a.mask[(size_t)(p.q0 + p.i0 + r) * a.mask_words + min(w, a.mask_words - 1)];
            g.m[k] = w < a.mask_words ? v : 0u;
        }
    }
    if (MOD && a.depth) {
#pragma unroll
        for (int k = 0; k < TreeStage<Sh>::D; ++k) {
            g.d[k] = a.depth[p.q0 + min(tid + k * Sh::THREADS, p.q.n - 1)];
        }
    }
}
template <bool MOD, class Sh, class A>
__device__ __forceinline__ void tree_stage_store(Sh& S, const TreeStage<Sh>& g, const A& a) {
    const int tid = (int)tree_fresh(threadIdx.x);
    if (a.mask) {
#pragma unroll
        for (int k = 0; k < TreeStage<Sh>::M; ++k)
            S.mask[(tid + k * Sh::THREADS) / kTreeMaskWords][tid % kTreeMaskWords] = g.m[k];
    }
    if (MOD && a.depth) {
#pragma unroll
        for (int k = 0; k < TreeStage<Sh>::D; ++k) S.depth[tid + k * Sh::THREADS] = tree_depth(g.d[k]);
    }
}

// The rows of a wave's tiles as B operands: column l16 of tile t is row first + 16 step t + l16 of the group (rows past it
// repeat its last), token i0 + row / G, head kvh G + row % G.
template <int NT>
struct TreeRows {
    pf16x8 q[NT][4];
    int pos[NT];       // the token's position relative to the context
    float slope[NT];
};
template <bool MOD, int NT, class A>
__device__ __forceinline__ void tree_load_rows(TreeRows<NT>& R, const A& a, const TreePiece& p, int kvh, int first, int step) {
    const int l16 = threadIdx.x & 15, lg = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = min(first + 16 * step * t + l16, p.rows - 1);
        const int i = r / a.G, h = kvh * a.G + (r - i * a.G);
        const size_t row = (size_t)(p.q0 + p.i0 + i) * a.Hq + h;
        const _Float16* qp = a.q + row * kHeadDim + 8 * lg;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) R.q[t][ks] = *reinterpret_cast<const pf16x8*>(qp + 32 * ks);
        R.pos[t] = MOD && a.depth ? tree_depth(a.depth[p.q0 + p.i0 + i]) : p.i0 + i;
        R.slope[t] = MOD && a.slopes ? a.slopes[h] * kTreeLog2e : 0.f;
        if (!MOD) dec_sign_q(R.q[t], a.scale_log2);
    }
}

// The sums so far of a wave's tiles: reference, sum over the lane's own keys, output.
template <int NT>
struct TreeState {
    float m[NT], l[NT];
    pf32x4 acc[NT][8];
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            m[t] = -INFINITY;
            l[t] = 0.f;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) acc[t][dt] = pf32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
};

// Raw products to scores in base 2: sm_scale and the cap. (Without either, the products stay and the softmax scales.)
template <bool MOD, int NT, int N>
__device__ __forceinline__ void tree_cap(float (&x)[NT][N]) {
    if constexpr (MOD) {
        const auto& h = *tree_args();
        const float cap_in = h.cap_in, cap_out = h.cap_out, scale_log2 = h.scale_log2;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (cap_out > 0.f) {   // (uniform)
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    x[t][e] *= cap_in;
                    top = fmaxf(top, fabsf(x[t][e]));
                }
                if (__builtin_amdgcn_ballot_w64(!(top <= 1.f))) {
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const float s = tree_tanh_small(x[t][e]), g = tree_tanh_large(x[t][e]);
                        x[t][e] = cap_out * (fabsf(x[t][e]) <= 1.f ? s : g);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < N; ++e) x[t][e] = cap_out * tree_tanh_small(x[t][e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) x[t][e] *= scale_log2;
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// The distance bias of keys that every row sees: x[t][4 y + j] is of key first[y] + j (relative to the context; the lane's
// four of a page).
template <bool MOD, int NA, int NT, int T>
__device__ __forceinline__ void tree_bias(float (&x)[NA][4 * T], const int (&first)[T], const TreeRows<NT>& R) {
    if constexpr (MOD) {
        if (tree_args()->slopes == nullptr) return;
#pragma unroll
        for (int y = 0; y < T; ++y)
#pragma unroll
            for (int t = 0; t < NA; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[t][4 * y + j] = fmaf(R.slope[t], (float)(first[y] + j - R.pos[t]), x[t][4 * y + j]);
    }
}

// The first n of a lane's four keys of a page, as bits.
__device__ __forceinline__ uint32_t tree_first(int n) { return (1u << min(max(n, 0), 4)) - 1u; }

// The same where the rows' masks, the window or the end of the keys cut through: scores of keys that a row does not see
// become -infinity. first[y]: the lane's first key of page y, at or past `end` for a page that is not there. Returns the
// keys that are there, as bits. (Bits by integer arithmetic: conditions would fill the scalar registers.)
template <bool MOD, int NT, int T, class Sh>
__device__ __forceinline__ uint32_t tree_see(float (&x)[NT][4 * T], const int (&first)[T], int end, int ctx, const TreeRows<NT>& R,
                                             const Sh& S, TreeCold cold, int tile0, int step) {
    const auto& f = *tree_args();
    const int gs = __builtin_ctz(f.G);   // G is a power of two
    const uint32_t masked = tree_fresh(f.mask ? ~0u : 0u);
    uint32_t real = 0u, near[NT];        // near: inside the window
#pragma unroll
    for (int y = 0; y < T; ++y) real |= tree_first(end - first[y]) << (4 * y);
#pragma unroll
    for (int t = 0; t < NT; ++t) near[t] = ~0u;
    if constexpr (MOD) {
        const int window = (int)tree_fresh((uint32_t)f.window);   // (in vector registers: the scalar ones are full)
        const bool deep = tree_fresh(f.depth ? 1u : 0u) != 0u;
        if (window > 0) {
            uint32_t kept = 0u;
#pragma unroll
            for (int y = 0; y < T; ++y) kept |= tree_first(f.sink - first[y]) << (4 * y);
#pragma unroll
            for (int t = 0; t < NT; ++t) near[t] = kept;
        }
#pragma unroll
        for (int e = 0; e < 4 * T; ++e) {
            const int at_key = tree_key_pos(deep, S, first[e >> 2] + (e & 3) - ctx);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int apart = R.pos[t] - at_key;
                near[t] |= (uint32_t)(apart - window) >> 31 << e;
                x[t][e] = fmaf(R.slope[t], (float)-apart, x[t][e]);   // (a slope of 0 without a bias)
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int tok = min(16 * (step * t + tile0) + (int)(tree_fresh(threadIdx.x) & 15u), cold.rows() - 1) >> gs;
        // of a mask four bits from drafted token j on (those before the first are cached keys, seen), of a chain the keys
        // up to the row's own; both, and one is taken (a branch costs the wide kernels more)
        uint32_t seen = 0u;
        const uint32_t* const row = S.mask[tok];
#pragma unroll
        for (int y = 0; y < T; ++y) {
            const int j = first[y] - ctx, w = j >> 5;
            const uint32_t lo = row[min(max(w, 0), kTreeMaskWords - 1)] | (uint32_t)(w >> 31);
            const uint32_t hi = row[min(max(w + 1, 0), kTreeMaskWords - 1)] | (uint32_t)((w + 1) >> 31);   // (past the last word: keys that are not there)
            const uint32_t tree = __builtin_amdgcn_alignbit(hi, lo, (uint32_t)j & 31u) & 15u;
            seen |= ((tree & masked) | (tree_first(cold.i0() + tok + 1 - j) & ~masked)) << (4 * y);
        }
        seen &= real & near[t];
#pragma unroll
        for (int e = 0; e < 4 * T; ++e) x[t][e] = seen >> e & 1u ? x[t][e] : -INFINITY;
        __builtin_amdgcn_sched_barrier(0);
    }
    return real;
}

// V elements of keys that are not there (bits of `real` from `at` on: the fragment's eight keys) become 0: they may hold
// anything, and 0 times NaN is NaN. Not 0 is returned if one that is there is not finite.
__device__ __forceinline__ uint32_t tree_keep(pf16x8& v, uint32_t real, int at) {
    pu32x4 u = __builtin_bit_cast(pu32x4, v);
    uint32_t odd = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        u[i] &= ((uint32_t)((int)(real << (31 - at - 2 * i)) >> 31) & 0xFFFFu) | ((uint32_t)((int)(real << (30 - at - 2 * i)) >> 31) & 0xFFFF0000u);
        odd |= tree_not_finite(u[i]);
    }
    v = __builtin_bit_cast(pf16x8, u);
    return tree_fresh(odd);   // (now, or every element waits in a register for the last)
}

// The online softmax, in base 2. A row's reference m is a score that is at most kTreeLag (in the exponent) below the
// largest yet: it, and with it the sum and the output, moves only when a block passes that. So most blocks need neither the
// maximum over a row's four lanes nor a rescaling (with the exact maximum: 8 x 8192 tokens, 64 drafted at G = 4, 113.5
// us against 102.5, the rescaling taken by about half of the blocks). A weight is exp2(score - m + kTreeShift), at most
// 2^15: fp16 holds it in full down to 2^-21 of the reference's weight and to within 2^-32 of it below; l, of the weights in
// 32 bits, carries the same factor. The weights enter the PV product rounded to fp16: with N(0, 1) values the
// output's error against 64 bits is 2.4e-4 of its norm, of which 2.1e-4 is its own rounding.
constexpr float kTreeLag = 8.f, kTreeShift = 7.f;
template <int N>
__device__ __forceinline__ float tree_largest(const float (&x)[N]) {
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) mx = fmaxf(mx, x[e]);
    return mx;
}
// The lag in scores (finite: -infinity plus it stays).
__device__ __forceinline__ float tree_slack(float scale2) { return fminf(kTreeLag / scale2, 1e38f); }
template <int NA, int NT, int N>
__device__ __forceinline__ void tree_softmax(const float (&x)[NA][N], TreeState<NT>& st, pf16x8 (&w)[NA][N / 8], float scale2, float slack) {
    bool grow = false;
#pragma unroll
    for (int t = 0; t < NA; ++t) grow |= tree_largest(x[t]) > st.m[t] + slack;
    if (__builtin_amdgcn_ballot_w64(grow)) {
#pragma unroll
        for (int t = 0; t < NA; ++t) {
            const float mn = fmaxf(st.m[t], col4_reduce<true>(tree_largest(x[t])));
            const float al = mn > st.m[t] ? __builtin_amdgcn_exp2f((st.m[t] - mn) * scale2) : 1.f;
            st.l[t] *= al;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) st.acc[t][dt] *= al;
            st.m[t] = mn;
        }
    }
#pragma unroll
    for (int t = 0; t < NA; ++t) {
        const float c = st.m[t] == -INFINITY ? kTreeShift : fmaf(-st.m[t], scale2, kTreeShift);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float pe = __builtin_amdgcn_exp2f(fmaf(x[t][e], scale2, c));
            st.l[t] += pe;
            w[t][e >> 3][e & 7] = (_Float16)pe;
        }
    }
}

// A piece row by row, for one thing alone: V of a key that some rows see and others do not holds NaN or infinity, which
// a product with the weight 0 of those others would pass on. A wave per row, 64 keys at a time: a key per lane for
// the scores, then two dims per lane, over the keys that the row sees.
template <bool MOD, class Sh>
__device__ __forceinline__ void tree_piece_rows(Sh& S, const TreePiece& p, int kvh, int end, TreeCold cold) {
    constexpr int ROWS = Sh::ROWS;
    const auto& a = *tree_args();
    const int wave = __builtin_amdgcn_readfirstlane(tree_fresh(threadIdx.x) >> 6), lane = (int)(tree_fresh(threadIdx.x) & 63u);
    const TreeSeq& sq = p.q;
    const int rows = cold.rows(), i0 = cold.i0(), q0 = cold.q0(), slot = cold.slot();
    float* const sp = reinterpret_cast<float*>(S.scratch(wave));          // the weights of 64 keys, then their pages
    int* const spg = reinterpret_cast<int*>(S.scratch(wave)) + 64;
    __syncthreads();   // the waves' outputs in the slots are given up
    for (int r = wave; r < rows; r += Sh::NW) {
        const int i = r / a.G, h = kvh * a.G + (r - i * a.G);
        const size_t row = (size_t)(q0 + i0 + i) * a.Hq + h;
        const _Float16* q = a.q + row * kHeadDim;
        const int pos = MOD && a.depth ? tree_depth(a.depth[q0 + i0 + i]) : i0 + i;
        const float slope = MOD && a.slopes ? a.slopes[h] * kTreeLog2e : 0.f;
        float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
        for (int at = p.p0; at < p.p1; at += 4) {   // four pages
            const int mine = at + (lane >> 4), page = sq.page(min(mine, p.p1 - 1)), key = page * kPage + (lane & 15), j = key - sq.ctx;
            bool seen = mine < p.p1 && key < end;
            if (seen && j >= 0) seen = a.mask ? (S.mask[i][min(j, kTreeMaxTokens - 1) >> 5] >> (j & 31) & 1u) != 0u : j <= i0 + i;
            const int apart = pos - (MOD ? tree_key_pos(a.depth != nullptr, S, j) : j);
            if (MOD && a.window > 0) seen = seen && (apart < a.window || key < a.sink);
            const int id = a.kv_indices[p.pb + page];
            float x = -INFINITY;
            if (seen) {
                const size_t off = ((size_t)(uint32_t)id * kPage + (key & 15)) * a.Hkv + kvh;
                const _Float16* k = reinterpret_cast<const _Float16*>(a.k) + off * kHeadDim;
                x = 0.f;
                for (int d = 0; d < kHeadDim; ++d) x = fmaf((float)q[d], (float)k[d], x);
                if (MOD && a.cap_out > 0.f) {
                    x *= a.cap_in;
                    x = a.cap_out * (fabsf(x) <= 1.f ? tree_tanh_small(x) : tree_tanh_large(x));
                } else {
                    x *= a.scale_log2;
                }
                if (MOD && a.slopes) x = fmaf(slope, (float)-apart, x);
            }
            float mx = x;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d, 64));
            const float mn = fmaxf(m, mx), al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            const float w = seen ? __builtin_amdgcn_exp2f(x - (mn == -INFINITY ? 0.f : mn)) : 0.f;
            if (m != -INFINITY) {   // (0 times what a row has summed of infinities would be NaN)
                l *= al;
                o0 *= al;
                o1 *= al;
            }
            m = mn;
            l += w;
            sp[lane] = w;
            spg[lane] = id;
            uint64_t todo = __builtin_amdgcn_ballot_w64(seen);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            while (todo) {
                const int e = __builtin_ctzll(todo);
                todo &= todo - 1;
                const size_t off = ((size_t)(uint32_t)spg[e] * kPage + (e & 15)) * a.Hkv + kvh;
                const _Float16* v = reinterpret_cast<const _Float16*>(a.v) + off * kHeadDim + 2 * lane;
                o0 = fmaf(sp[e], (float)v[0], o0);
                o1 = fmaf(sp[e], (float)v[1], o1);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d, 64);
        const float inv = l == 0.f ? 0.f : 1.f / l, lse = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * kTreeLn2;
        if (slot < 0) {
            a.out[row * kHeadDim + 2 * lane] = (_Float16)(o0 * inv);
            a.out[row * kHeadDim + 2 * lane + 1] = (_Float16)(o1 * inv);
            if (lane == 0) a.lse[row] = lse;
        } else {
            const size_t pr = (size_t)slot * ROWS + r;
            *reinterpret_cast<float2*>(a.part_o + pr * kHeadDim + 2 * lane) = make_float2(o0 * inv, o1 * inv);
            if (lane == 0) a.part_lse[pr] = lse;
        }
    }
}

// ---- few rows: the key-split body -------------------------------------------------------------------
//
// Bound by HBM: up to 16 NT rows are on each key. A wave's 16 KB slot is read into registers whole (one tile; K, then V,
// with two) and filled again while the block is computed; two workgroups a CU. 32 ragged sequences of 200-6000 tokens,
// one capped token each at G = 4: 223 MB in 42 us and the merge's 4, where a plain read of as much takes 33.

// A block's operands from the wave's slot, as dec_read_block (of which they are the halves).
__device__ __forceinline__ void tree_read_k(DecBlock& b, uint8_t* slot, int l16, int lg) {
    typedef __attribute__((address_space(3))) uint8_t lds_u8;
    const uint32_t kl = tree_fresh((uint32_t)(l16 * 256 + ((((l16 >> 2) << 2) | (lg ^ (l16 & 3))) << 4)));
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
            b.k[t][ks] = __builtin_bit_cast(pf16x8, *(const __attribute__((address_space(3))) pu32x4*)(
                                                        (lds_u8*)slot + ((kl ^ (uint32_t)(ks << 6)) + kDecPageBytes * t)));
}
__device__ __forceinline__ void tree_read_v(DecBlock& b, uint8_t* slot, int l16, int lg) {
    typedef __attribute__((address_space(3))) uint8_t lds_u8;
    const int key = 4 * lg + (l16 >> 2);
    const uint32_t vl = tree_fresh((uint32_t)(2 * kDecPageBytes + key * 256 + ((((key & 7) << 1) | ((l16 & 3) >> 1)) << 4) + 8 * (l16 & 1)));
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
        pf16x4 half[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
            half[h] = __builtin_bit_cast(pf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                (__attribute__((address_space(3))) lds_f16x4*)((lds_u8*)slot + ((vl ^ (uint32_t)(dt << 5)) + kDecPageBytes * h))));
        b.v[dt] = pf16x8{half[0][0], half[0][1], half[0][2], half[0][3], half[1][0], half[1][1], half[1][2], half[1][3]};
    }
}

// The lane offsets of a page's loads: row n = 4 i + lg of a page, LDS position l16 of it: chunk l16 ^ n of K, l16 ^ ((n & 7)
// << 1) of V (the swizzles that dec_read_block reads), from the bases of row lg, ^ i << 6 and ^ (i & 1) << 7, + i rows4.
struct TreeOffsets {
    uint32_t k, v, rows4;
    __device__ __forceinline__ TreeOffsets(int Hkv, int l16, int lg)
        : k((uint32_t)(lg * Hkv * 256 + ((l16 ^ lg) << 4))), v((uint32_t)(lg * Hkv * 256 + ((l16 ^ (lg << 1)) << 4))),
          rows4((uint32_t)(4 * Hkv * 256)) {}
};
__device__ __forceinline__ void tree_dma_k(const uint8_t* page, uint32_t base, uint32_t rows4, uint32_t lds) {
#pragma unroll
    for (int i = 0; i < 4; ++i) dec_dma(page, (base ^ (uint32_t)(i << 6)) + i * rows4, lds + 1024 * i);
}
__device__ __forceinline__ void tree_dma_v(const uint8_t* page, uint32_t base, uint32_t rows4, uint32_t lds) {
#pragma unroll
    for (int i = 0; i < 4; ++i) dec_dma(page, (base ^ (uint32_t)((i & 1) << 7)) + i * rows4, lds + 1024 * i);
}

template <int NT, bool MOD>
__device__ __forceinline__ void tree_piece(TreeSplitShared<NT>& S, const TreePiece& p, int kvh, TreeCold cold) {
    typedef TreeSplitShared<NT> SH;
    constexpr int ROWS = 16 * NT;
    const auto& a = *tree_args();
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int l16 = lane & 15, lg = lane >> 4;
    const TreeSeq& sq = p.q;
    const int ctx = sq.ctx;

    __syncthreads();   // the piece before is done with the LDS
    if (tid == 0) S.wild[p.par ^ 1] = 0;   // the next piece's
    PD_STAMP(2 + 8 * p.par);

    const TreeKeys ks = tree_keys<MOD>(a, p, lane);
    const int end = ks.end, p1 = ks.p1;
    const TreeOrder o = tree_order(p.p0 + 2 * wave, 8, 2, p1, ks.a0, ks.a1);

    const uint32_t page_bytes = (uint32_t)(kPage * a.Hkv * 256);
    const TreeOffsets off(a.Hkv, l16, lg);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)S.slot[wave];
    const uint8_t* const kc = a.k + kvh * 256;
    const uint8_t* const vc = a.v + kvh * 256;
    // lane 2 x + y holds page y of the x-th block of a window of 32
    int pidv = 0;
    auto load_ids = [&](int i) {
        const int at = p.p0 + 8 * o.block(min(i + (lane >> 1), o.n - 1)) + 2 * wave + (lane & 1);
        pidv = tree_args()->kv_indices[p.pb + sq.page(min(at, p1 - 1))];
    };
    auto issue = [&](int n) {
        if (n >= o.n) return;
        const int at = p.p0 + 8 * o.block(n) + 2 * wave;
        const uint32_t kb = tree_fresh(off.k), vb = tree_fresh(off.v);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            if (at + y >= p1) break;
            const size_t page = (size_t)(uint32_t)__builtin_amdgcn_readlane(pidv, 2 * (n & 31) + y) * page_bytes;
            tree_dma_k(kc + page, kb, off.rows4, lds0 + kDecPageBytes * y);
            tree_dma_v(vc + page, vb, off.rows4, lds0 + kDecPageBytes * (2 + y));
        }
    };

    // The page ids, then the q and mask rows on the way, then the first block's loads as soon as the ids are there
    if (o.n > 0) load_ids(0);
    TreeRows<NT> R;
    tree_load_rows<MOD>(R, a, p, kvh, 0, 1);
    const bool drafts = p1 > p.p0 && (sq.page(p1 - 1) + 1) * kPage > ctx;   // (uniform) the piece holds drafted keys
    TreeStage<SH> stage;
    if (drafts) tree_stage_load<MOD>(stage, a, p);
    if (o.n > 0) issue(0);
    PD_STAMP(3 + 8 * p.par);
    if (drafts) tree_stage_store<MOD>(S, stage, a);
    uint32_t wild = 0u;   // not 0: an element of V, of a key that not every row may see, is not finite
    TreeState<NT> st;
    st.reset();
    // (a scale of 0 would make an unseen key's -inf a NaN)
    const float scale2 = MOD ? 1.f : a.scale_log2 == 0.f ? 0x1p-126f : fabsf(a.scale_log2), slack = tree_slack(scale2);

    auto block = [&](int n, auto EDGE) {
        constexpr bool edge = decltype(EDGE)::value;
        // One tile: all operands to registers, and the next block's loads are on their way before any arithmetic. Two
        // tiles: K first, V after the scores, in the registers of K.
        DecBlock b;
        dec_wait_loads();
        tree_read_k(b, S.slot[wave], l16, lg);
        if constexpr (NT == 1) tree_read_v(b, S.slot[wave], l16, lg);
        dec_wait_lds();
        auto next = [&]() {
            if (((n + 1) & 31) == 0 && n + 1 < o.n) load_ids(n + 1);
            issue(n + 1);
        };
        if constexpr (NT == 1) next();

        const int at = p.p0 + 8 * o.block(n) + 2 * wave;
        float x[NT][8];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                pf32x4 c0 = pf32x4{0.f, 0.f, 0.f, 0.f}, c1 = c0;
                c0 = mfma16x16x32(b.k[y][0], R.q[t][0], c0);
                c1 = mfma16x16x32(b.k[y][1], R.q[t][1], c1);
                c0 = mfma16x16x32(b.k[y][2], R.q[t][2], c0);
                c1 = mfma16x16x32(b.k[y][3], R.q[t][3], c1);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[t][4 * y + j] = c0[j] + c1[j];
            }
        if constexpr (NT > 1) {
            __builtin_amdgcn_sched_barrier(0);
            tree_read_v(b, S.slot[wave], l16, lg);
            dec_wait_lds();
            next();
        }
        tree_cap<MOD>(x);
        if constexpr (edge) {
            const int lg4 = (int)(tree_fresh(lane) >> 4) * 4;
            const int first[2] = {sq.page(at) * kPage + lg4, (at + 1 < p1 ? sq.page(at + 1) * kPage : end) + lg4};
            const uint32_t real = tree_see<MOD>(x, first, end, ctx, R, S, cold, 0, 1);
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) wild |= tree_keep(b.v[dt], real, 0);
        } else {
            const int first[2] = {sq.page(at) * kPage + 4 * lg - ctx, sq.page(at + 1) * kPage + 4 * lg - ctx};
            tree_bias<MOD>(x, first, R);
        }
        pf16x8 w[NT][1];
        tree_softmax(x, st, w, scale2, slack);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
#pragma unroll
            for (int t = 0; t < NT; ++t) st.acc[t][dt] = mfma16x16x32(b.v[dt], w[t][0], st.acc[t][dt]);
    };

    if (drafts) __syncthreads();   // mask rows and depths
    PD_STAMP(4 + 8 * cold.flag());
    for (int n = 0; n < o.plain; ++n) block(n, std::false_type{});
    for (int n = o.plain; n < o.n; ++n) block(n, std::true_type{});
    PD_STAMP(5 + 8 * cold.flag());

    // Join of the four waves: each leaves its output in its slot (row r's four dims c at place c ^ r of the row, so
    // that the 16 rows of a store lie in different banks).
    dec_wait_lds();
    if (__builtin_amdgcn_ballot_w64(wild != 0u) && lane == 0) S.wild[cold.flag()] = 1;
    float* const so = reinterpret_cast<float*>(S.slot[wave]);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float L = col4_reduce<false>(st.l[t]);
        if (lg == 0) {
            S.m[wave][16 * t + l16] = st.m[t];
            S.l[wave][16 * t + l16] = L;
        }
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
            *reinterpret_cast<pf32x4*>(so + ((16 * t + l16) * 32 + ((4 * dt + lg) ^ l16)) * 4) = st.acc[t][dt];
    }
    __syncthreads();
    const auto& f = *tree_args();
    const int kvh_ = (int)tree_fresh_s(blockIdx.x) % f.Hkv;
    if (S.wild[cold.flag()]) {   // (uniform)
        tree_piece_rows<MOD>(S, p, kvh_, end, cold);
        return;
    }
    const int rows = cold.rows(), slot = cold.slot(), token0 = cold.q0() + cold.i0();
#pragma unroll 1
    for (int it = 0; it < ROWS * 32 / kTreeThreads; ++it) {
        const int idx = it * kTreeThreads + (int)tree_fresh(threadIdx.x), r = idx >> 5, c = idx & 31;
        if (r >= rows) continue;
        float mw[kTreeWaves], M = -INFINITY, L = 0.f;
        pf32x4 O = pf32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kTreeWaves; ++w) {
            mw[w] = S.m[w][r];
            M = fmaxf(M, mw[w]);
        }
#pragma unroll
        for (int w = 0; w < kTreeWaves; ++w) {
            const float al = mw[w] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw[w] - M) * scale2);
            const pf32x4 v = *reinterpret_cast<const pf32x4*>(reinterpret_cast<const float*>(S.slot[w]) + (r * 32 + (c ^ (r & 15))) * 4);
            L = fmaf(al, S.l[w][r], L);
#pragma unroll
            for (int j = 0; j < 4; ++j) O[j] = fmaf(al, v[j], O[j]);
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const float lse = L == 0.f ? -INFINITY : fmaf(M, scale2, __builtin_amdgcn_logf(L) - kTreeShift) * kTreeLn2;
        if (slot < 0) {
            const int i = r / f.G;
            const size_t row = (size_t)(token0 + i) * f.Hq + kvh_ * f.G + (r - i * f.G);
            const pf16x4 h = {(_Float16)(O[0] * inv), (_Float16)(O[1] * inv), (_Float16)(O[2] * inv), (_Float16)(O[3] * inv)};
            *reinterpret_cast<pf16x4*>(f.out + row * kHeadDim + 4 * c) = h;
            if (c == 0) f.lse[row] = lse;
        } else {
            const size_t row = (size_t)slot * ROWS + r;
            *reinterpret_cast<pf32x4*>(f.part_o + row * kHeadDim + 4 * c) = O * inv;
            if (c == 0) f.part_lse[row] = lse;
        }
    }
}

// ---- many rows: the row-split body -----------------------------------------------------------------
//
// With 32 rows on each key the key-split body is bound by the bytes that its waves wait for (8 x 8192 tokens, 64
// drafted at G = 4: 203 us, 338 TFLOP/s): every row group streams all K and V again. Here a workgroup holds 16 NT rows in
// each of NW waves, and all waves read the same 64-key blocks, staged by direct loads. No join at the end.
//
// Four waves, two workgroups a CU: two LDS buffers, one block ahead; a barrier a block; the two workgroups' phases drift
// apart, so that one's softmax meets the other's MFMAs (8 x 8192, 64 drafted: 99.0 us; a chain of 512 on 2 x 8192: 159).
//
// Eight waves, one workgroup a CU: half the bytes for the same rows, four buffers, two blocks ahead. Each SIMD has one wave
// of the first four and one of the others, and a step between two barriers is for the first: PV product of block i - 1,
// scores and softmax of block i; for the others: softmax and PV product of block i - 1, scores of block i. So each step
// starts with one wave's MFMAs beside the other's vector work (96.3 and 155.7 us; all waves in the first order 98.2 and 161.0;
// two workgroups of four waves 97.7 and 162.0).
template <int NW, int NT, bool MOD>
__device__ __forceinline__ void tree_piece_wide(TreeWideShared<NW, NT>& S, const TreePiece& p, int kvh, TreeCold cold) {
    typedef TreeWideShared<NW, NT> SH;
    typedef __attribute__((address_space(3))) uint8_t lds_u8;
    constexpr int ROWS = SH::ROWS, NB = SH::NB, AHEAD = NB / 2;   // blocks ahead
    const auto& a = *tree_args();
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int l16 = lane & 15, lg = lane >> 4;
    const TreeSeq& sq = p.q;
    const int ctx = sq.ctx;

    __syncthreads();   // the piece before is done with the LDS
    if (tid == 0) S.wild[p.par ^ 1] = 0;   // the next piece's
    PD_STAMP(2 + 8 * p.par);

    const TreeKeys ks = tree_keys<MOD>(a, p, lane);
    const int end = ks.end, p1 = ks.p1;
    const TreeOrder o = tree_order(p.p0, 4, 4, p1, ks.a0, ks.a1);

    // Staging: wave w moves page w % 4 of every block, of four waves K and V, of eight K (the first four) or V.
    const int pg = wave & 3;
    const uint32_t page_bytes = (uint32_t)(kPage * a.Hkv * 256);
    const TreeOffsets off(a.Hkv, l16, lg);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)S.block[0] + kDecPageBytes * pg;
    const uint8_t* const kc = a.k + kvh * 256;
    const uint8_t* const vc = a.v + kvh * 256;
    int pidv = 0;   // lane x: this wave's page of the x-th block of a window of 64
    auto load_ids = [&](int n) {
        const int at = p.p0 + 4 * o.block(min(n + lane, o.n - 1)) + pg;
        pidv = tree_args()->kv_indices[p.pb + sq.page(min(at, p1 - 1))];
    };
    auto loads = [&](int n) { return n < o.n && p.p0 + 4 * o.block(n) + pg < p1; };   // whether block n has a page for this wave
    auto issue = [&](int n) {
        if ((n & 63) == 0 && n > 0 && n < o.n) load_ids(n);
        if (!loads(n)) return;
        const uint32_t kb = tree_fresh(off.k), vb = tree_fresh(off.v);
        const size_t page = (size_t)(uint32_t)__builtin_amdgcn_readlane(pidv, n & 63) * page_bytes;
        const uint32_t lds = lds0 + (n & (NB - 1)) * kTreeBlockBytes;
        if (NW == 4 || wave < 4) tree_dma_k(kc + page, kb, off.rows4, lds);
        if (NW == 4 || wave >= 4) tree_dma_v(vc + page, vb, off.rows4, lds + kTreeBlockBytes / 2);
    };
    // This wave's loads of block n are done; those of the block after it may still be on their way.
    auto arrived = [&](int n) {
        if (NW == 8 && loads(n + 1)) {
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        } else {
            dec_wait_loads();
        }
    };

    if (o.n > 0) load_ids(0);
    // Tile t of wave w is tile NW t + w of the group's rows (so that few rows fill the first tiles of all waves).
    TreeRows<NT> R;
    tree_load_rows<MOD>(R, a, p, kvh, 16 * wave, NW);
    const bool drafts = p1 > p.p0 && (sq.page(p1 - 1) + 1) * kPage > ctx;   // (uniform) the piece holds drafted keys
    TreeStage<SH> stage;
    if (drafts) tree_stage_load<MOD>(stage, a, p);
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) issue(n);
    PD_STAMP(3 + 8 * p.par);
    if (drafts) tree_stage_store<MOD>(S, stage, a);
    uint32_t wild = 0u;   // as in tree_piece
    TreeState<NT> st;
    st.reset();
    const float scale2 = MOD ? 1.f : a.scale_log2 == 0.f ? 0x1p-126f : fabsf(a.scale_log2), slack = tree_slack(scale2);

    auto buffer = [&](int n) { return (lds_u8*)S.block[0] + (n & (NB - 1)) * kTreeBlockBytes; };
    // S^T: x[t][4 tk + j] = product of key 16 tk + 4 lg + j and row l16 of tile t; K of tile tk + 1 is read before the MFMAs
    // of tile tk (but in an edge block, whose bits take the registers)
    auto scores = [&](int n, auto& x, auto EDGE) {
        constexpr int NA = sizeof(x) / sizeof(x[0]);
        constexpr int ahead = decltype(EDGE)::value ? 0 : 1;
        lds_u8* const buf = buffer(n);
        const uint32_t kl = tree_fresh((uint32_t)(l16 * 256 + ((((l16 >> 2) << 2) | (lg ^ (l16 & 3))) << 4)));
        auto kfrag = [&](int tk, pf16x8 (&ka)[4]) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
                ka[ks] = __builtin_bit_cast(pf16x8, *(const __attribute__((address_space(3))) pu32x4*)(
                                                        buf + ((kl ^ (uint32_t)(ks << 6)) + kDecPageBytes * tk)));
        };
        pf16x8 ka[1 + ahead][4];
        if (ahead) kfrag(0, ka[0]);
#pragma unroll
        for (int tk = 0; tk < 4; ++tk) {
            if (tk < 4 - ahead) kfrag(tk + ahead, ka[(tk + ahead) & ahead]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < NA; ++t) {
                pf32x4 c = pf32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) c = mfma16x16x32(ka[tk & ahead][ks], R.q[t][ks], c);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[t][4 * tk + j] = c[j];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto first_key = [&](int n, int tk) {
        const int at = p.p0 + 4 * o.block(n) + tk;
        return at < p1 ? sq.page(at) * kPage : end;
    };
    // Products to weights
    auto weights = [&](int n, auto& x, auto& w, auto EDGE) {
        tree_cap<MOD>(x);
        const int lg4 = (int)(tree_fresh(lane) >> 4) * 4;
        int first[4];
        if constexpr (decltype(EDGE)::value) {
#pragma unroll
            for (int tk = 0; tk < 4; ++tk) first[tk] = first_key(n, tk) + lg4;
            (void)tree_see<MOD>(x, first, end, ctx, R, S, cold, wave, NW);
        } else if constexpr (MOD) {
#pragma unroll
            for (int tk = 0; tk < 4; ++tk) first[tk] = sq.page(p.p0 + 4 * o.block(n) + tk) * kPage + lg4 - ctx;
            tree_bias<MOD>(x, first, R);
        }
        tree_softmax(x, st, w, scale2, slack);
    };
    // O^T += V^T P^T; V of dim tile dt + 1 is read before the MFMAs of dt (but in an edge block)
    auto product = [&](int n, const auto& w, auto EDGE) {
        constexpr int NA = sizeof(w) / sizeof(w[0]);
        constexpr bool edge = decltype(EDGE)::value;
        constexpr int ahead = edge ? 0 : 1;
        lds_u8* const buf = buffer(n) + kTreeBlockBytes / 2;
        uint32_t real = 0u;
        if constexpr (edge) {
            const int lg4 = (int)(tree_fresh(lane) >> 4) * 4;
#pragma unroll
            for (int tk = 0; tk < 4; ++tk) real |= tree_first(end - first_key(n, tk) - lg4) << (4 * tk);
        }
        const int vk = 4 * lg + (l16 >> 2);
        const uint32_t vl = tree_fresh((uint32_t)(vk * 256 + ((((vk & 7) << 1) | ((l16 & 3) >> 1)) << 4) + 8 * (l16 & 1)));
        auto vfrag = [&](int dt, int h) {
            pf16x4 half[2];
#pragma unroll
            for (int y = 0; y < 2; ++y)
                half[y] = __builtin_bit_cast(pf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                    (__attribute__((address_space(3))) lds_f16x4*)(buf + ((vl ^ (uint32_t)(dt << 5)) + kDecPageBytes * (2 * h + y)))));
            return pf16x8{half[0][0], half[0][1], half[0][2], half[0][3], half[1][0], half[1][1], half[1][2], half[1][3]};
        };
        pf16x8 va[1 + ahead][2];
        if (ahead) {
            va[0][0] = vfrag(0, 0);
            va[0][1] = vfrag(0, 1);
        }
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            if (dt < 8 - ahead) {
                va[(dt + ahead) & ahead][0] = vfrag(dt + ahead, 0);
                va[(dt + ahead) & ahead][1] = vfrag(dt + ahead, 1);
            }
            if constexpr (edge) {
#pragma unroll
                for (int h = 0; h < 2; ++h) wild |= tree_keep(va[dt & ahead][h], real, 8 * h);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < NA; ++t) st.acc[t][dt] = mfma16x16x32(va[dt & ahead][h], w[t][h], st.acc[t][dt]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    if (o.n > 0) arrived(0);
    __syncthreads();   // mask rows, depths, the first block
    PD_STAMP(4 + 8 * cold.flag());
    if constexpr (NW == 4) {
        auto block = [&](int n, auto EDGE, auto TILES) {
            constexpr int NA = decltype(TILES)::value;
            // Of two workgroups on a CU the one that came first issues first, and would be done a quarter sooner (76 and 97
            // us of 8 x 8192 tokens, 64 drafted); the other one goes first in every second block (102.5 -> 99.0 us; a
            // chain of 512 on 2 x 8192 164 -> 159).
            if (cold.late()) {
                if (n & 1) __builtin_amdgcn_s_setprio(1);
                else __builtin_amdgcn_s_setprio(0);
            }
            issue(n + 1);
            float x[NA][16];
            pf16x8 w[NA][2];
            scores(n, x, EDGE);
            weights(n, x, w, EDGE);
            product(n, w, EDGE);
            arrived(n + 1);
            dec_barrier();
        };
        // A wave whose second tile has no row leaves it out (32 ragged contexts, 5-27 drafted tokens at G = 8, so groups of
        // 8-128 rows: 77.7 -> 75.0 us)
        const std::integral_constant<int, NT> all{};
        const std::integral_constant<int, 1> one{};
        int n = 0;
        if (NT == 1 || cold.rows() > 16 * (NW + wave)) {
            for (; n < o.plain; ++n) block(n, std::false_type{}, all);
        } else {
            for (; n < o.plain; ++n) block(n, std::false_type{}, one);
        }
        for (; n < o.n; ++n) block(n, std::true_type{}, all);
    } else if (o.n > 0) {
        // Steps 0 .. n: the step in which both of a wave's blocks are plain is the loop; the others are the general one.
        const std::false_type plain{};
        const std::true_type edge{};
        auto done = [&](int i) {
            arrived(i + 1);
            dec_barrier();
        };
        if (wave < 4) {
            pf16x8 w[NT][2];
            for (int i = 0; i <= o.n;) {
                issue(i + 2);
                if (i > 0) product(i - 1, w, edge);
                if (i < o.n) {
                    float x[NT][16];
                    scores(i, x, edge);
                    weights(i, x, w, edge);
                }
                done(i);
                for (++i; i < o.plain; ++i) {
                    issue(i + 2);
                    __builtin_amdgcn_s_setprio(1);   // (the wave at its MFMAs first: 157.0 -> 155.7 us)
                    product(i - 1, w, plain);
                    float x[NT][16];
                    scores(i, x, plain);
                    __builtin_amdgcn_s_setprio(0);
                    weights(i, x, w, plain);
                    done(i);
                }
            }
        } else {
            float x[NT][16];
            const int last = min(o.plain, o.n - 1);
            for (int i = 0; i <= o.n;) {
                issue(i + 2);
                if (i > 0) {
                    pf16x8 w[NT][2];
                    weights(i - 1, x, w, edge);
                    product(i - 1, w, edge);
                }
                if (i < o.n) scores(i, x, edge);
                done(i);
                for (++i; i <= last; ++i) {
                    issue(i + 2);
                    pf16x8 w[NT][2];
                    weights(i - 1, x, w, plain);
                    __builtin_amdgcn_s_setprio(1);
                    product(i - 1, w, plain);
                    scores(i, x, plain);
                    __builtin_amdgcn_s_setprio(0);
                    done(i);
                }
            }
        }
    }
    PD_STAMP(5 + 8 * cold.flag());

    if (__builtin_amdgcn_ballot_w64(wild != 0u) && lane == 0) S.wild[cold.flag()] = 1;
    __syncthreads();
    const auto& f = *tree_args();
    const int kvh_ = (int)tree_fresh_s(blockIdx.x) % f.Hkv;
    if (S.wild[cold.flag()]) {   // (uniform)
        tree_piece_rows<MOD>(S, p, kvh_, end, cold);
        return;
    }
    const int rows = cold.rows(), slot = cold.slot(), token0 = cold.q0() + cold.i0();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float L = col4_reduce<false>(st.l[t]), m = st.m[t];
        const int r = 16 * (NW * t + wave) + (int)(tree_fresh(lane) & 15u);
        if (r >= rows) continue;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        const float lse = L == 0.f ? -INFINITY : fmaf(m == -INFINITY ? 0.f : m, scale2, __builtin_amdgcn_logf(L) - kTreeShift) * kTreeLn2;
        if (slot < 0) {
            const int i = r / f.G;
            const size_t row = (size_t)(token0 + i) * f.Hq + kvh_ * f.G + (r - i * f.G);
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) {
                const pf32x4 v = st.acc[t][dt] * inv;
                *reinterpret_cast<pf16x4*>(f.out + row * kHeadDim + 16 * dt + 4 * lg) =
                    pf16x4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
            }
            if (lg == 0) f.lse[row] = lse;
        } else {
            const size_t row = (size_t)slot * ROWS + r;
#pragma unroll
            for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<pf32x4*>(f.part_o + row * kHeadDim + 16 * dt + 4 * lg) = st.acc[t][dt] * inv;
            if (lg == 0) f.part_lse[row] = lse;
        }
    }
}

// A workgroup's range, piece by piece.
template <class Sh, class Piece>
__device__ __forceinline__ void tree_workgroup(const TreeArgs& a, Sh& S, Piece piece) {
    // timestamps (timeline build only), the last two pieces': 0 start, 1 the range found; with par the piece's flag, 2 + 8
    // par begun, 3 + 8 par the first loads issued, 4 + 8 par at the first block, 5 + 8 par the blocks done, 6 + 8 par
    // written; 31 end
    PD_STAMP(0);
    const int g = blockIdx.x / a.Hkv, kvh = blockIdx.x - g * a.Hkv;
    if (threadIdx.x == 0) S.wild[0] = 0;
    TreeRange r;
    if (!tree_find_range<Sh::NW>(a, S.scan, g, r)) {
        if (kvh == 0 && threadIdx.x == 0) a.cuts[g] = make_int4(0, 0, 0, 0);
        return;
    }
    PD_STAMP(1);
    // The first item, the units of it before the range, and (kv head 0) what the merge has to know: an item that
    // the boundary before this range cuts, which of its cuts that is, and its pieces.
    const int lane = threadIdx.x & 63;
    int b = r.b, left = r.left, j, skip;
    int half = 0, entries = lane == 25 ? r.extra : r.entries;   // (half: the entries that hold sequence b's)
    auto entry = [&](int i) { return __builtin_amdgcn_readlane(entries, half + i); };
    auto sequence = [&](const auto& k) { return tree_seq_of(k, entry(0), entry(1), entry(2), entry(3), entry(4), __builtin_amdgcn_readlane(entries, 25)); };
    {
        const auto& k = *tree_args();
        const TreeSeq t = sequence(k);
        j = __builtin_amdgcn_readfirstlane(t.group_of(r.in));
        skip = __builtin_amdgcn_readfirstlane((int)(r.in - t.before(j)));
        if (kvh == 0 && threadIdx.x == 0) {
            const int64_t first = r.lo - skip;
            const int g0 = r.cuts.of(first + t.extra), g1 = r.cuts.of(first + t.last_unit(j)), i0 = j << k.tl;
            k.cuts[g] = make_int4(max(entry(3), 0) + i0, min(1 << k.tl, t.n - i0) * k.G, g0 < g && g <= g1 ? g1 - g0 + 1 : 0, g - g0 - 1);
        }
    }
    int par = 0;
    while (left > 0) {
        TreePiece p;
        const auto& k = *tree_args();
        p.q = sequence(k);
        p.pb = entry(0);
        p.q0 = max(entry(3), 0);
        if (j >= p.q.groups) {
            if (++b >= k.B) break;   // (not reached: the units of the items from here on are at least `left`)
            j = 0;
            const int x = (int)tree_fresh((uint32_t)lane), v = tree_load_entry(k, b + 1, x);
            entries = (x & 24) == half ? v : entries;
            half ^= 8;
            continue;
        }
        const int take = min(left, p.q.units(j) - skip), f0 = p.q.first_page(j, skip), f1 = p.q.first_page(j, skip + take);
        left -= take;
        skip = 0;
        if (f0 >= f1) {   // no page's first unit: before the item's first or behind its last
            ++j;
            continue;
        }
        p.i0 = j << k.tl;
        p.tokens = min(1 << k.tl, p.q.n - p.i0);
        p.rows = p.tokens * k.G;
        p.p0 = f0;
        p.p1 = min(f1, p.q.attended());
        const int s = tree_slot(f0, f1, p.q.pages(j));
        p.slot = s < 0 ? -1 : 2 * (int)tree_fresh_s(blockIdx.x) + s;
        p.par = par;
        ++j;
        par ^= 1;
        // (the loop's own state is kept in lanes of the entries' register meanwhile)
        const uint32_t x = tree_fresh((uint32_t)lane);
        entries = x < 16 || x > 24 ? entries : x == 16 ? left : x == 17 ? b : x == 18 ? j : x == 19 ? half | par
                : x == 20 ? p.i0 : x == 21 ? p.rows : x == 22 ? p.q0 : x == 23 ? p.slot : (int)((int)tree_fresh_s(blockIdx.x) * 2 >= k.ranges * k.Hkv);
        entries = (int)tree_fresh((uint32_t)entries);
        piece(p, kvh, entries);
        left = __builtin_amdgcn_readlane(entries, 16);
        b = __builtin_amdgcn_readlane(entries, 17);
        j = __builtin_amdgcn_readlane(entries, 18);
        half = __builtin_amdgcn_readlane(entries, 19) & 8;
        par = __builtin_amdgcn_readlane(entries, 19) & 1;
        PD_STAMP(6 + 8 * (par ^ 1));
    }
    PD_STAMP(31);
}

template <int NT, bool MOD>
__global__ __launch_bounds__(kTreeThreads, 2) void tree_split_kernel(TreeArgs a) {
    __shared__ TreeSplitShared<NT> S;
    tree_workgroup(a, S, [&](const TreePiece& p, int kvh, int cold) { tree_piece<NT, MOD>(S, p, kvh, {cold}); });
}
template <int NW, int NT, bool MOD>
__global__ __launch_bounds__(64 * NW, 2) void tree_wide_kernel(TreeArgs a) {
    __shared__ TreeWideShared<NW, NT> S;
    static_assert(8 / NW * sizeof(S) <= 160 * 1024, "eight waves on a CU");
    tree_workgroup(a, S, [&](const TreePiece& p, int kvh, int cold) { tree_piece_wide<NW, NT, MOD>(S, p, kvh, {cold}); });
}

// Merge of the cut items. Boundary g, kv head: of the item that it cuts (pieces n: cut cut.w of n - 1) every (n - 1)-th
// row. A row's output is formed by one half of a wave, four dims a lane, from its pieces in their order.
// Few pieces (as of many rows): a half takes a row, its pieces' loads ahead of the arithmetic. Many (as of one
// long context): a workgroup takes a row, its eight halves every eighth piece each, joined in the halves' order.
struct TreeMerged {
    float m = -INFINITY, w = 0.f;
    pf32x4 o = pf32x4{0.f, 0.f, 0.f, 0.f};
    __device__ __forceinline__ void add(float lse, const pf32x4& v) {
        if (lse == -INFINITY) return;
        const float mn = fmaxf(m, lse);
        const float sc = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * kTreeLog2e);
        const float e = __builtin_amdgcn_exp2f((lse - mn) * kTreeLog2e);
        w = fmaf(w, sc, e);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(e, v[j], o[j] * sc);
        m = mn;
    }
    __device__ __forceinline__ void write(const TreeArgs& a, const int4& cut, int kvh, int r, int c) const {
        const float inv = w == 0.f ? 0.f : 1.f / w;
        const int i = r / a.G;
        const size_t row = (size_t)(cut.x + i) * a.Hq + kvh * a.G + (r - i * a.G);
        // (not through the L2, which is written back at the kernel's end: chain of 512 on 2 x 8192 150.3 -> 149.4 us)
        __builtin_nontemporal_store(pf16x4{(_Float16)(o[0] * inv), (_Float16)(o[1] * inv), (_Float16)(o[2] * inv), (_Float16)(o[3] * inv)},
                                    reinterpret_cast<pf16x4*>(a.out + row * kHeadDim + 4 * c));
        if (c == 0) a.lse[row] = w == 0.f ? -INFINITY : fmaf(__builtin_amdgcn_logf(w), kTreeLn2, m == -INFINITY ? 0.f : m);
    }
};

__global__ __launch_bounds__(kTreeThreads) void tree_merge_kernel(TreeArgs a, int ROWS) {
    const int g = blockIdx.x / a.Hkv + 1, kvh = blockIdx.x % a.Hkv;
    const int4 cut = a.cuts[g];
    const int n = cut.z, g0 = g - 1 - cut.w;
    if (n == 0) return;
    const int tid = threadIdx.x, half = tid >> 5, c = tid & 31;
    const int mine = (cut.y - cut.w + n - 2) / (n - 1);   // rows of this boundary: cut.w + (n - 1) x, x < mine
    // piece k: range g0 + k, slot 1 of the first's workgroup, slot 0 of the others'
    auto slot = [&](int k) { return ((size_t)((g0 + k) * a.Hkv + kvh) * 2 + (k == 0)) * ROWS; };
    constexpr int U = 4;   // pieces at a time
    if (n <= 2 * U) {
        for (int x = (int)blockIdx.y * 8 + half; x < mine; x += 8 * (int)gridDim.y) {
            const int r = cut.w + (n - 1) * x;
            TreeMerged t;
            for (int k0 = 0; k0 < n; k0 += U) {
                float l[U];
                pf32x4 v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (k0 + u >= n) break;   // (uniform)
                    const size_t s = slot(k0 + u) + r;
                    l[u] = a.part_lse[s];
                    v[u] = *reinterpret_cast<const pf32x4*>(a.part_o + s * kHeadDim + 4 * c);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (k0 + u >= n) break;
                    t.add(l[u], v[u]);
                }
            }
            t.write(a, cut, kvh, r, c);
        }
        return;
    }
    __shared__ float s_m[8], s_w[8];
    __shared__ pf32x4 s_o[8][32];
    for (int x = blockIdx.y; x < mine; x += gridDim.y) {
        const int r = cut.w + (n - 1) * x;
        TreeMerged t;
        for (int k0 = half; k0 - half < n; k0 += 8 * U) {
            float l[U];
            pf32x4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t s = slot(min(k0 + 8 * u, n - 1)) + r;
                l[u] = a.part_lse[s];
                v[u] = *reinterpret_cast<const pf32x4*>(a.part_o + s * kHeadDim + 4 * c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (k0 + 8 * u < n) t.add(l[u], v[u]);
        }
        if (c == 0) {
            s_m[half] = t.m;
            s_w[half] = t.w;
        }
        s_o[half][c] = t.o;
        __syncthreads();
        if (half == 0) {
            TreeMerged J;
#pragma unroll
            for (int h = 0; h < 8; ++h) J.m = fmaxf(J.m, s_m[h]);
#pragma unroll
            for (int h = 0; h < 8; ++h) {
                const float s = s_m[h] == -INFINITY ? (s_w[h] == 0.f ? 0.f : s_w[h]) : __builtin_amdgcn_exp2f((s_m[h] - J.m) * kTreeLog2e);   // (s_w: NaN)
                J.w = fmaf(s_w[h], s, J.w);
                const pf32x4 ho = s_o[h][c];
#pragma unroll
                for (int j = 0; j < 4; ++j) J.o[j] = fmaf(ho[j], s, J.o[j]);
            }
            J.write(a, cut, kvh, r, c);
        }
        __syncthreads();
    }
}

template <int NT>
void launch_tree_split(const TreeArgs& a, bool mod, hipStream_t s) {
    const int W = a.ranges * a.Hkv;
    if (mod) tree_split_kernel<NT, true><<<W, kTreeThreads, 0, s>>>(a);
    else tree_split_kernel<NT, false><<<W, kTreeThreads, 0, s>>>(a);
}
template <int NW, int NT>
void launch_tree_wide(const TreeArgs& a, bool mod, hipStream_t s) {
    const int W = a.ranges * a.Hkv;
    if (mod) tree_wide_kernel<NW, NT, true><<<W, 64 * NW, 0, s>>>(a);
    else tree_wide_kernel<NW, NT, false><<<W, 64 * NW, 0, s>>>(a);
}

}  // namespace

hipError_t launch_tree_attention(const TreeArgs& a, hipStream_t s) {
    if (a.n_tokens <= 0 || a.B <= 0 || a.ranges <= 0) return hipSuccess;
    const bool mod = a.cap_out > 0.f || a.slopes || a.window > 0;
    if (a.rows == 16) launch_tree_split<1>(a, mod, s);
    else if (a.rows == 32) launch_tree_split<2>(a, mod, s);
    else if (a.rows == 64) launch_tree_wide<4, 1>(a, mod, s);
    else if (a.rows == 128) launch_tree_wide<4, 2>(a, mod, s);
    else if (a.rows == 256 && !mod) tree_wide_kernel<8, 2, false><<<a.ranges * a.Hkv, 64 * 8, 0, s>>>(a);
    else return hipErrorInvalidValue;
    if (a.ranges > 1) {
        const int most = std::min(a.rows, std::max(1, a.max_tokens) * a.G);
        // (eight rows a workgroup, a half wave each)
        tree_merge_kernel<<<dim3((a.ranges - 1) * a.Hkv, (most + 7) / 8), kTreeThreads, 0, s>>>(a, a.rows);
    }
    return hipGetLastError();
}

}  // namespace pdattn
