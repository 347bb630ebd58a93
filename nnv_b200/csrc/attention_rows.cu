// Attention of few positions over many states: up to eight rows (sixteen for 16-bit types) of positions times query heads
// that share a state head, the single-token step of a decoder first of all.  Bound by reading K and V once.
//
// A cluster of blocks shares the states of one state head.  Their warps take blocks of states in turn and keep their own
// running maximum, sum and output for all rows, so K and V are read once for the whole group of heads.  The warps'
// results meet in shared memory, the blocks' in distributed shared memory, always in the same order: one launch, no
// workspace, no atomics.
//
// 16-bit types: a warp copies its blocks of 16 states through a ring of its own (cp.async, a few KB in flight per warp
// whatever the arithmetic does) and multiplies with warp-wide mma.sync: rows fill one 16-row tile, tcgen05's smallest has
// 64 or 128, and at this bound its rate would not show.  Products with the FMA pipe took 50 instructions a state, which
// was the bound; these take 6.  Weights enter P V as the sum of two 16-bit values, because a few rows' rounding errors do
// not average out: with up to eight rows the second value rides in the tile's idle rows.  In fp16 they carry a factor 2^14,
// so that those below 2^-14 keep their bits too.
//
// float and double: states go straight into registers, products run on the FMA pipe with two terms an instruction.
//
// 64 x 1 x 4096, 32 heads over 8 of 128 channels, bf16, lengths at random: 480 MB of valid states in 85 us,
// 5.65 TB/s (0.86 of a copy; 6.5 TB/s with equal lengths).
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "attention.cuh"
#include "mma_f64.cuh"

namespace cg = cooperative_groups;

namespace nnvb {
namespace {

constexpr int WARPS = 4, ROWS_THREADS = WARPS * 32;

// The batch entry with the i-th most states, by counting, for up to ROWS_THREADS entries: blocks that run one after the
// other end together when the long ones start first (64 x 1 x 4096 x 8 x 4 x 128 bf16, lengths at random: 98 us in
// the batch's order, 85 so).  Counting takes a block a microsecond, so entries have to be long (120 x 1 x 200 x 8 x 64: 21, 26).
__device__ int by_length(const AttnArgs& a, int i) {
    __shared__ int len[ROWS_THREADS], entry;
    const int t = threadIdx.x;
    if (t < a.B) len[t] = attn_len(a, t);
    __syncthreads();
    if (t < a.B) {
        int before = 0;
        for (int j = 0; j < a.B; ++j) before += len[j] > len[t] || (len[j] == len[t] && j < t);
        if (before == i) entry = t;
    }
    __syncthreads();
    return entry;
}

template <typename T, int R, int DP>
struct RowsShape {
    using A = typename AccOf<T>::type;
    static constexpr int E = 16 / sizeof(T);                       // elements of a 16-byte piece
    static constexpr int PIECES = DP / E;                          // pieces of a state
    static constexpr int KEYS = 32 / sizeof(T);                    // states of a block
    // lanes that share a state in Q K^T: the rows' channels of a lane fill at most 64 registers
    static constexpr int WANT = (R <= 2 ? 4 : R * 2) * (sizeof(T) == 8 ? 2 : 1);
    static constexpr int LK = WANT < PIECES ? WANT : PIECES;
    static constexpr int KSUB = 32 / LK;                           // states at once
    static constexpr int STEPS = KEYS / KSUB;
    static constexpr int PL = PIECES / LK;                         // pieces of a lane
    // P V: a lane has CPL pieces of every KP-th state
    static constexpr int CPL = PIECES > 32 ? PIECES / 32 : 1;
    static constexpr int KP = PIECES < 32 ? 32 / PIECES : 1;
    static constexpr int VL = KEYS / KP;
    static_assert(KEYS % KSUB == 0 && PIECES % LK == 0 && KEYS % KP == 0, "");
};

template <typename T, int R, int DP>
__global__ void __launch_bounds__(ROWS_THREADS)
attn_rows_kernel(AttnArgs a) {
    using S = RowsShape<T, R, DP>;
    using A = typename S::A;
    using P = Pack<T, S::E>;
    constexpr int E = S::E;
    __shared__ __align__(16) A ps[WARPS][S::KEYS][R];              // scores, then weights
    __shared__ A fs[WARPS][R];
    __shared__ __align__(16) A part_o[WARPS][R][DP];
    __shared__ A part_m[WARPS][R], part_l[WARPS][R];
    __shared__ __align__(16) A all_o[R][DP];                       // the block's result, read by the cluster
    __shared__ A all_m[R], all_l[R];

    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), world = int(cluster.num_blocks());
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int unit = int(blockIdx.x) / world;                       // batch entry and state head
    const int g = unit % a.Hkv, b = a.longest_first ? by_length(a, unit / a.Hkv) : unit / a.Hkv;
    const int G = a.Hq / a.Hkv, rows = G * a.Lq;
    const int n = attn_len(a, b);
    const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + g * a.ks[2];
    const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + g * a.vs[2];
    const A ninf = -INFINITY;

    // rows' channels of this lane, times scale log2 e
    A q[R][S::PL * E];
    const int sub = lane % S::LK, kin = lane / S::LK;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const T* qr = static_cast<const T*>(a.q) + b * a.qs[0] + int64_t(r / G) * a.qs[1] + int64_t(g * G + r % G) * a.qs[2];
#pragma unroll
        for (int j = 0; j < S::PL; ++j) {
            const int d = (sub + S::LK * j) * E;
            P v;
            const bool in = r < rows && d < a.D;
            if (in) v = *reinterpret_cast<const P*>(qr + d);
#pragma unroll
            for (int e = 0; e < E; ++e) q[r][j * E + e] = in ? to_acc(v.v[e]) * A(a.scale * LOG2E) : A(0);
        }
    }
    A o[R][S::CPL * E];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int e = 0; e < S::CPL * E; ++e) o[r][e] = 0;
    // softmax: a lane has state lane % KEYS of a block for rows lane / KEYS, + HALVES, ...
    constexpr int HALVES = 32 / S::KEYS, RL = (R + HALVES - 1) / HALVES;
    const int key = lane % S::KEYS, row0 = lane / S::KEYS;
    A m[RL], l[RL];
#pragma unroll
    for (int i = 0; i < RL; ++i) { m[i] = ninf; l[i] = 0; }

    const int blocks = (n + S::KEYS - 1) / S::KEYS, stride = world * WARPS;
    P kb[S::STEPS * S::PL], vb[S::VL * S::CPL];
    auto load_k = [&](int blk) {
#pragma unroll
        for (int s = 0; s < S::STEPS; ++s) {
            const int j = blk * S::KEYS + s * S::KSUB + kin;
#pragma unroll
            for (int i = 0; i < S::PL; ++i) {
                const int d = (sub + S::LK * i) * E;
                if (j < n && d < a.D) kb[s * S::PL + i] = *reinterpret_cast<const P*>(kp + int64_t(j) * a.ks[1] + d);
                else
#pragma unroll
                    for (int e = 0; e < E; ++e) kb[s * S::PL + i].v[e] = from_acc<T, A>(A(0));
            }
        }
    };
    const int piece = lane % (S::PIECES < 32 ? S::PIECES : 32), kgrp = lane / (S::PIECES < 32 ? S::PIECES : 32);
    auto load_v = [&](int blk) {
#pragma unroll
        for (int s = 0; s < S::VL; ++s) {
            const int j = blk * S::KEYS + s * S::KP + kgrp;
#pragma unroll
            for (int i = 0; i < S::CPL; ++i) {
                const int d = (piece + 32 * i) * E;
                if (j < n && d < a.D) vb[s * S::CPL + i] = *reinterpret_cast<const P*>(vp + int64_t(j) * a.vs[1] + d);
                else
#pragma unroll
                    for (int e = 0; e < E; ++e) vb[s * S::CPL + i].v[e] = from_acc<T, A>(A(0));
            }
        }
    };
    int blk = rank * WARPS + warp;
    if (blk < blocks) load_k(blk);
    for (; blk < blocks; blk += stride) {
        load_v(blk);
#pragma unroll
        for (int s = 0; s < S::STEPS; ++s) {
            Pair<A> acc[R];
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r] = both(A(0));
#pragma unroll
            for (int i = 0; i < S::PL; ++i)
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const P& x = kb[s * S::PL + i];
                    const Pair<A> kk{A(to_acc(x.v[e])), A(to_acc(x.v[e + 1]))};
#pragma unroll
                    for (int r = 0; r < R; ++r) acc[r] = fma2(Pair<A>{q[r][i * E + e], q[r][i * E + e + 1]}, kk, acc[r]);
                }
            A v[R];
#pragma unroll
            for (int r = 0; r < R; ++r) v[r] = across(acc[r]);
            // sum over the LK lanes: while a lane holds several rows it hands half of them to its partner
            int row = 0, count = R;
#pragma unroll
            for (int w = S::LK / 2; w > 0; w >>= 1) {
                if (count > 1) {
                    const int half = count / 2;
                    const bool up = sub & w;
#pragma unroll
                    for (int r = 0; r < R / 2; ++r)
                        if (r < half) {
                            const A give = up ? v[r] : v[r + half], mine = up ? v[r + half] : v[r];
                            v[r] = mine + __shfl_xor_sync(0xffffffffu, give, w, 32);
                        }
                    if (up) row += half;
                    count = half;
                } else {
                    v[0] += __shfl_xor_sync(0xffffffffu, v[0], w, 32);
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (r < count) ps[warp][s * S::KSUB + kin][row + r] = v[r];
        }
        if (blk + stride < blocks) load_k(blk + stride);
        __syncwarp();
        const bool in = blk * S::KEYS + key < n;
        bool moved = false;
#pragma unroll
        for (int i = 0; i < RL; ++i) {
            const int r = row0 + i * HALVES;
            const A s = in && r < R ? ps[warp][key][r < R ? r : 0] : ninf;
            A mx = s;
#pragma unroll
            for (int w = S::KEYS / 2; w > 0; w >>= 1) {
                const A y = __shfl_xor_sync(0xffffffffu, mx, w, 32);
                mx = y > mx ? y : mx;
            }
            const A mn = mx > m[i] ? mx : m[i], base = mn == ninf ? A(0) : mn;
            const A f = exp_acc(m[i] - base), p = in ? exp_acc(s - base) : A(0);
            if (mn != m[i]) moved = true;
            m[i] = mn;
            l[i] = l[i] * f + p;
            if (r < R) {
                ps[warp][key][r] = p;
                if (key == 0) fs[warp][r] = f;
            }
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const A f = fs[warp][r];
#pragma unroll
                for (int e = 0; e < S::CPL * E; ++e) o[r][e] *= f;
            }
        }
#pragma unroll
        for (int s = 0; s < S::VL; ++s) {
            const auto p = *reinterpret_cast<const Pack<A, R>*>(&ps[warp][s * S::KP + kgrp][0]);
#pragma unroll
            for (int i = 0; i < S::CPL; ++i)
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const P& x = vb[s * S::CPL + i];
                    const Pair<A> vv{A(to_acc(x.v[e])), A(to_acc(x.v[e + 1]))};
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const Pair<A> y = fma2(both(p.v[r]), vv, Pair<A>{o[r][i * E + e], o[r][i * E + e + 1]});
                        o[r][i * E + e] = y.x;
                        o[r][i * E + e + 1] = y.y;
                    }
                }
        }
        __syncwarp();                      // the scores' places are free
    }

    // ---- the warps' results -------------------------------------------------------------------------------------------
#pragma unroll
    for (int i = 0; i < RL; ++i) {
        const int r = row0 + i * HALVES;
#pragma unroll
        for (int w = S::KEYS / 2; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w, 32);
        if (r < R && key == 0) { part_m[warp][r] = m[i]; part_l[warp][r] = l[i]; }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < S::CPL; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                A x = o[r][i * E + e];
#pragma unroll
                for (int w = S::PIECES; w < 32; w *= 2) x += __shfl_xor_sync(0xffffffffu, x, w, 32);
                if (kgrp == 0) part_o[warp][r][(piece + 32 * i) * E + e] = x;
            }
    __syncthreads();
    for (int i = threadIdx.x; i < R * DP; i += ROWS_THREADS) {
        const int r = i / DP, d = i % DP;
        A top = ninf, sum = 0, x = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = part_m[w][r] > top ? part_m[w][r] : top;
        const A base = top == ninf ? A(0) : top;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const A f = exp_acc(part_m[w][r] - base);
            sum += part_l[w][r] * f;
            x += part_o[w][r][d] * f;
        }
        all_o[r][d] = x;
        if (d == 0) { all_m[r] = top; all_l[r] = sum; }
    }
    cluster.sync();
    // ---- the blocks' results: every block writes its share of the channels ------------------------------------------------
    for (int i = rank * ROWS_THREADS + threadIdx.x; i < rows * DP; i += world * ROWS_THREADS) {
        const int r = i / DP, d = i % DP;
        A top = ninf, sum = 0, x = 0;
        for (int w = 0; w < world; ++w) {
            const A y = *cluster.map_shared_rank(&all_m[r], w);
            top = y > top ? y : top;
        }
        const A base = top == ninf ? A(0) : top;
        for (int w = 0; w < world; ++w) {
            const A f = exp_acc(*cluster.map_shared_rank(&all_m[r], w) - base);
            sum += *cluster.map_shared_rank(&all_l[r], w) * f;
            x += *cluster.map_shared_rank(&all_o[r][d], w) * f;
        }
        const int tok = r / G, h = g * G + r % G;
        if (d < a.D)
            static_cast<T*>(const_cast<void*>(a.o))[b * a.os[0] + tok * a.os[1] + h * a.os[2] + d] =
                from_acc<T, A>(n > 0 ? x / sum : A(0));
        if (d == 0 && a.lse)
            static_cast<A*>(a.lse)[(int64_t(b) * a.Hq + h) * a.Lq + tok] = n > 0 ? top / A(LOG2E) + log_acc(sum) : ninf;
    }
    cluster.sync();                        // nobody leaves while its shared memory is read
}

// ---------------------------------------------------------------------------
// 16-bit types

template <typename T> __device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// four 8 x 8 tiles; lane i gives the address of row i % 8 of tile i / 8
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}


// blocks of states of a warp's ring: as many as let several blocks share an SM
template <int DP> constexpr int ROWS_RING = DP == 64 ? 4 : 3;

// WIDE: 9 to 16 rows; else up to 8
template <typename T, int DP, bool WIDE>
__global__ void __launch_bounds__(ROWS_THREADS)
attn_rows_mma_kernel(AttnArgs a) {
    constexpr int KEYS = 16, ROW = DP * 2, BLOCK = KEYS * ROW;     // bytes of a state, of a block of states of K or V
    constexpr int PIECES = DP / 8, NR = WIDE ? 16 : 8, NT = DP / 8, KS = DP / 16, RING = ROWS_RING<DP>;
    extern __shared__ __align__(128) unsigned char rings[];
    __shared__ float part_m[WARPS][NR], part_l[WARPS][NR], all_m[NR], all_l[NR];
    __shared__ __align__(16) float all_o[NR][DP];

    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), world = int(cluster.num_blocks());
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, gr = lane / 4, tq = lane % 4;
    const int unit = int(blockIdx.x) / world;
    const int g = unit % a.Hkv, b = a.longest_first ? by_length(a, unit / a.Hkv) : unit / a.Hkv;
    const int G = a.Hq / a.Hkv, rows = G * a.Lq;
    const int n = attn_len(a, b);
    const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + g * a.ks[2];
    const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + g * a.vs[2];
    unsigned char* ring = rings + warp * RING * 2 * BLOCK;
    const uint32_t ring_at = smem_u32(ring);
    const float c = float(a.scale * LOG2E);
    constexpr float SHIFT = std::is_same<T, __half>::value ? 14.f : 0.f;

    const int blocks = (n + KEYS - 1) / KEYS, stride = world * WARPS, first = rank * WARPS + warp;
    // block `blk` into stage s; states behind the valid ones and channels behind the last become 0
    auto load = [&](int blk, int s) {
        if (blk < blocks) {
#pragma unroll
            for (int i = 0; i < KEYS * PIECES / 32; ++i) {
                const int at = i * 32 + lane, j = at / PIECES, p = at % PIECES;
                const int64_t tok = blk * KEYS + j;
                const int bytes = tok < n && p * 8 < a.D ? 16 : 0;
                const int64_t at_tok = bytes ? tok : 0;
                const int d = bytes ? p * 8 : 0;
                unsigned char* dst = ring + s * 2 * BLOCK + j * ROW + ((p ^ (j & 7)) * 16);
                cp_async16(dst, kp + at_tok * a.ks[1] + d, bytes);
                cp_async16(dst + BLOCK, vp + at_tok * a.vs[1] + d, bytes);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < RING - 1; ++s) load(first + s * stride, s);

    uint32_t q[KS][4];
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = gr + (i & 1) * 8, d = k * 16 + tq * 2 + (i / 2) * 8;
            q[k][i] = 0;
            if (r < rows && d < a.D)
                q[k][i] = *reinterpret_cast<const uint32_t*>(static_cast<const T*>(a.q) + b * a.qs[0] + int64_t(r / G) * a.qs[1] +
                                                             int64_t(g * G + r % G) * a.qs[2] + d);
        }
    float o[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    constexpr int NH = WIDE ? 2 : 1;                               // rows of a lane: gr, gr + 8
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    int s = 0;
    for (int blk = first; blk < blocks; blk += stride) {
        load(blk + (RING - 1) * stride, s == 0 ? RING - 1 : s - 1);
        cp_async_wait<RING - 1>();
        __syncwarp();
        const uint32_t kat = ring_at + s * 2 * BLOCK, vat = kat + BLOCK;
        float sc[2][4] = {};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            uint32_t f[4];
            const int j = (lane / 16) * 8 + lane % 8, p = k * 2 + lane / 8 % 2;
            ldmatrix4(f, kat + j * ROW + ((p ^ (j & 7)) * 16));
            mma_16816<T>(sc[0], q[k], f[0], f[1]);
            mma_16816<T>(sc[1], q[k], f[2], f[3]);
        }
        const int rest = n - blk * KEYS;
        float p[2][4];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& x = sc[t][h * 2 + e];
                    x = t * 8 + tq * 2 + e < rest ? x * c : -INFINITY;
                    mx = fmaxf(mx, x);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1, 32));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2, 32));
            const float mn = fmaxf(m[h], mx), base = mn == -INFINITY ? 0.f : mn;
            const float f = exp2f(m[h] - base);
            if (__any_sync(0xffffffffu, mn != m[h])) {
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    o[i][h * 2] *= f;
                    o[i][h * 2 + 1] *= f;
                    if (!WIDE) { o[i][2] *= f; o[i][3] *= f; }
                }
            }
            m[h] = mn;
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    p[t][h * 2 + e] = t * 8 + tq * 2 + e < rest ? exp2f(sc[t][h * 2 + e] - base + SHIFT) : 0.f;
                    sum += p[t][h * 2 + e];
                }
            l[h] = l[h] * f + sum;
        }
        // weights as two 16-bit values
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h >= NH) continue;
                const T x = from_acc<T, float>(p[t][h * 2]), y = from_acc<T, float>(p[t][h * 2 + 1]);
                const T u = from_acc<T, float>(p[t][h * 2] - to_acc(x)), w = from_acc<T, float>(p[t][h * 2 + 1] - to_acc(y));
                Pack<T, 2> ph{{x, y}}, pl{{u, w}};
                hi[t * 2 + h] = *reinterpret_cast<uint32_t*>(&ph);
                lo[t * 2 + h] = *reinterpret_cast<uint32_t*>(&pl);
            }
        if (!WIDE) { hi[1] = lo[0]; hi[3] = lo[2]; }
#pragma unroll
        for (int i = 0; i < NT; i += 2) {
            uint32_t f[4];
            const int j = (lane / 8 % 2) * 8 + lane % 8, pc = i + lane / 16;
            ldmatrix4_trans(f, vat + j * ROW + ((pc ^ (j & 7)) * 16));
            mma_16816<T>(o[i], hi, f[0], f[1]);
            mma_16816<T>(o[i + 1], hi, f[2], f[3]);
            if (WIDE) {
                mma_16816<T>(o[i], lo, f[0], f[1]);
                mma_16816<T>(o[i + 1], lo, f[2], f[3]);
            }
        }
        __syncwarp();                      // the stage is free
        if (++s == RING) s = 0;
    }
    cp_async_wait<0>();

    // ---- the warps' results: over the rings, a warp its own ---------------------------------------------------------------
    __syncwarp();
    float* mine = reinterpret_cast<float*>(ring);                  // [NR][DP]
#pragma unroll
    for (int h = 0; h < NH; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1, 32);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2, 32);
        if (tq == 0) { part_m[warp][gr + h * 8] = m[h]; part_l[warp][gr + h * 8] = l[h]; }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                mine[(gr + h * 8) * DP + i * 8 + tq * 2 + e] = WIDE ? o[i][h * 2 + e] : o[i][e] + o[i][2 + e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < NR * DP; i += ROWS_THREADS) {
        const int r = i / DP, d = i % DP;
        float top = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, part_m[w][r]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = exp2f(part_m[w][r] - base);
            sum += part_l[w][r] * f;
            x += reinterpret_cast<const float*>(rings + w * RING * 2 * BLOCK)[i] * f;
        }
        all_o[r][d] = x;
        if (d == 0) { all_m[r] = top; all_l[r] = sum; }
    }
    cluster.sync();
    // ---- the blocks' results: every block writes its share of the channels ------------------------------------------------
    for (int i = rank * ROWS_THREADS + threadIdx.x; i < rows * DP; i += world * ROWS_THREADS) {
        const int r = i / DP, d = i % DP;
        float top = -INFINITY, sum = 0.f, x = 0.f;
        for (int w = 0; w < world; ++w) top = fmaxf(top, *cluster.map_shared_rank(&all_m[r], w));
        const float base = top == -INFINITY ? 0.f : top;
        for (int w = 0; w < world; ++w) {
            const float f = exp2f(*cluster.map_shared_rank(&all_m[r], w) - base);
            sum += *cluster.map_shared_rank(&all_l[r], w) * f;
            x += *cluster.map_shared_rank(&all_o[r][d], w) * f;
        }
        const int tok = r / G, h = g * G + r % G;
        if (d < a.D)
            static_cast<T*>(const_cast<void*>(a.o))[b * a.os[0] + tok * a.os[1] + h * a.os[2] + d] =
                from_acc<T, float>(n > 0 ? x / sum : 0.f);
        if (d == 0 && a.lse)
            static_cast<float*>(a.lse)[(int64_t(b) * a.Hq + h) * a.Lq + tok] = n > 0 ? (top - SHIFT) / float(LOG2E) + logf(sum) : -INFINITY;
    }
    cluster.sync();                        // nobody leaves while its shared memory is read
}

// Blocks per state head: a power of two (others leave SMs of a cluster's group idle: 8 x 2 x 4096 x 8 x 2 x 128 float, 74 us with 8,
// 90 with 6) up to 16, at least two blocks of states a warp, and at most a third more blocks than `per_sm` an SM: more
// would run as a second round (16 x 1 x 2048 x 8 x 4 x 128 bf16: 36 us with 4, 30 with 2).  Sixteen blocks with a large ring
// take most of a group of SMs, so few such clusters run at once (18 x 1 x 4096 x 1 x 8 x 128 bf16: 27 us with 16, 19 with 8).
template <typename K>
int launch_rows(K kernel, cudaStream_t st, const AttnArgs& a, int keys, int per_sm, int smem) {
    const int64_t units = int64_t(a.B) * a.Hkv;
    const int64_t sms = sm_count(), blocks = sms * per_sm * 4 / 3, most = ceil_div(a.Lk, keys * WARPS * 2);
    int world = 1;
    while (world < (smem > 64 * 1024 && units * 16 > sms ? 8 : 16) && world < most && units * world * 2 <= blocks) world *= 2;
    NNVB_REQUIRE(units * world < (int64_t(1) << 31), "nnvb_cross_attention_forward: too many state heads (%lld) for one launch",
                 (long long)units);
    if (world > 8) NNVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (smem > 48 * 1024) NNVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(units * world));
    cfg.blockDim = dim3(ROWS_THREADS);
    cfg.dynamicSmemBytes = size_t(smem);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = unsigned(world);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    AttnArgs args = a;
    args.longest_first = a.lengths && a.B > 1 && a.B <= ROWS_THREADS && a.Lk >= 16 * a.B && units * world > sms * per_sm;
    NNVB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args));
    return NNVB_OK;
}

template <typename T, int DP>
int rows_by_count(cudaStream_t st, const AttnArgs& a) {
    const int64_t rows = int64_t(a.Hq / a.Hkv) * a.Lq;
    if constexpr (sizeof(T) == 2) {
        constexpr int SMEM = WARPS * ROWS_RING<DP> * 2 * 16 * DP * 2;
        return rows <= 8 ? launch_rows(attn_rows_mma_kernel<T, DP, false>, st, a, 16, 2, SMEM)
                         : launch_rows(attn_rows_mma_kernel<T, DP, true>, st, a, 16, 2, SMEM);
    } else {
        constexpr int KEYS = RowsShape<T, 1, DP>::KEYS;
        if (rows <= 1) return launch_rows(attn_rows_kernel<T, 1, DP>, st, a, KEYS, 3, 0);
        if (rows <= 2) return launch_rows(attn_rows_kernel<T, 2, DP>, st, a, KEYS, 3, 0);
        if (rows <= 4) return launch_rows(attn_rows_kernel<T, 4, DP>, st, a, KEYS, 3, 0);
        return launch_rows(attn_rows_kernel<T, 8, DP>, st, a, KEYS, 3, 0);
    }
}
template <typename T>
int rows_by_head(cudaStream_t st, const AttnArgs& a) {
    return a.D <= 64 ? rows_by_count<T, 64>(st, a) : rows_by_count<T, 128>(st, a);
}

}  // namespace

bool attn_rows_takes(const AttnArgs& a) {
    const int64_t e = dtype_bytes(a.dtype);
    if (int64_t(a.Hq / a.Hkv) * a.Lq > (e == 2 ? 16 : 8) || a.D > 128 || a.D * e % 16) return false;
    for (auto* s : {a.qs, a.ks, a.vs})
        for (int i = 0; i < 3; ++i)
            if (s[i] * e % 16) return false;
    for (const void* p : {a.q, a.k, a.v})
        if (reinterpret_cast<uintptr_t>(p) % 16) return false;
    return true;
}

int attn_forward_rows(cudaStream_t st, const AttnArgs& a) {
    switch (a.dtype) {
        case NNVB_F64: return rows_by_head<double>(st, a);
        case NNVB_F32: return rows_by_head<float>(st, a);
        case NNVB_BF16: return rows_by_head<__nv_bfloat16>(st, a);
        default: return rows_by_head<__half>(st, a);
    }
}

}  // namespace nnvb
