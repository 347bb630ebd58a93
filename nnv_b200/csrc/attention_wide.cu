// Attention over an encoder's states for float and double tensors with head sizes up to 128.
//
// Forward.  A block of four warps takes 64 rows, positions of the query heads that share a state head, and walks over
// tiles of states with the running maximum and sum of each row's softmax.  K and V tiles arrive by cp.async in a buffer
// each: V while the scores are computed, the next K while the weights meet V.  Products stop at the head's channels.
//   double  tensor cores (mma.sync f64 m16n8k8): a warp has 16 rows.  The order of the contraction is free, so channels
//           (and states) 2t, 2t+1 take the places t, t+4 of a lane: operands are loaded 16 bytes at a time, and scores
//           become weights in the registers they are in.  Bound by the FP64 pipe.
//   float   FMA pipe, two terms an instruction: 8 x 16 threads with 8 x 4 scores each; 12 16-byte loads feed 128 FMAs, half
//           of the cycles the FMAs take.  Bound by the FMA pipe.
// Two or three blocks an SM hide part of each other's exponentials and hand-overs: 36 TFLOP/s in float and 16 in double at
// 8 x 1024 x 2048 x 16 x 64 and 8 x 512 x 1024 x 8 x 64, half of what the pipes give; with 128 channels registers and shared
// memory hold fewer, 31 and 13.  Backward: 26 and 13 TFLOP/s, 20 and 8 with 128 channels.
// Where 64-row tiles give the GPU too few blocks, or do not come out even, a cluster of up to 16 blocks shares the states
// of a tile; their results meet in distributed shared memory in a fixed order.
#include <cooperative_groups.h>

#include <algorithm>

#include "attention.cuh"
#include "mma_f64.cuh"

namespace cg = cooperative_groups;

namespace nnvb {
namespace {

constexpr int BQ = 64, THREADS = 128;

// Row strides (elements) that spread the loads of a warp over all banks.
template <typename T, int DP, int BK_ = 0>
struct WideShape {
    static constexpr bool F64 = sizeof(T) == 8;
    static constexpr int BK = BK_ ? BK_ : (F64 && DP == 128 ? 32 : 64);        // states of a tile (backward: rows streamed)
    static constexpr int LDQ = F64 ? DP + 8 : DP + 4, LDK = LDQ, LDV = F64 ? DP + 2 : DP + 4, LDP = BK + 4;
    static constexpr int NQ = BQ * LDQ, NK = BK * LDK, NV = BK * LDV, NP = F64 ? 0 : BQ * LDP;
    static constexpr int BYTES = (NQ + NK + NV + NP) * int(sizeof(T));
};

// rows r0 .. r0 + ROWS; rows from n_rows on and columns from D on become 0.  at(r): where row r begins, in elements from g.
// vec: asynchronous
template <typename T, int ROWS, int DP, int LD, typename At>
__device__ __forceinline__ void load_rows(T* s, const T* g, At&& at, int r0, int n_rows, int D, bool vec) {
    constexpr int V = 16 / sizeof(T), P = DP / V;
    if (vec) {
#pragma unroll 4
        for (int i = threadIdx.x; i < ROWS * P; i += THREADS) {
            const int r = i / P, c = i % P * V;
            const bool in = r0 + r < n_rows && c < D;              // D is a multiple of V
            cp_async16(s + r * LD + c, g + (in ? at(r0 + r) + c : 0), in ? 16 : 0);
        }
    } else {
        for (int i = threadIdx.x; i < ROWS * DP; i += THREADS) {
            const int r = i / DP, c = i % DP;
            s[r * LD + c] = r0 + r < n_rows && c < D ? g[at(r0 + r) + c] : T(0);
        }
    }
    cp_async_commit();
}

// A warp's or thread's part of the tile: scores and output of its rows.  Row of index i, and the type's products.
template <typename T, int DP, int BK = 0> struct Work;

template <int DP, int BK_>
struct Work<double, DP, BK_> {
    using S = WideShape<double, DP, BK_>;
    static constexpr int NR = 2, NT = S::BK / 8;                   // rows of a lane; 8-state tiles
    double s[NT][4], o[DP / 8][4];
    int warp, g, t;
    __device__ __forceinline__ Work() : warp(threadIdx.x / 32), g(threadIdx.x % 32 / 4), t(threadIdx.x % 4) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = 0;
    }
    __device__ __forceinline__ int row(int i) const { return warp * 16 + g + i * 8; }
    // rest: states of the tile that count; 8-state tiles behind them are left out, and channels from D on
    template <int LDY = S::LDK>
    __device__ __forceinline__ void scores(const double* Q, const double* K, int rest, int D) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] = 0;
        const double* q = Q + row(0) * S::LDQ + 2 * t;
        const double* k = K + g * LDY + 2 * t;
#pragma unroll 4
        for (int d = 0; d < DP; d += 8) {
            if (d >= D) break;
            const double2 x = *reinterpret_cast<const double2*>(q + d), y = *reinterpret_cast<const double2*>(q + 8 * S::LDQ + d);
            const double a[4] = {x.x, y.x, x.y, y.y};
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                if (j * 8 >= rest) break;
                const double2 z = *reinterpret_cast<const double2*>(k + j * 8 * LDY + d);
                const double b[2] = {z.x, z.y};
                dmma_16x8x8(s[j], a, b);
            }
        }
    }
    // f(row index, state of the tile, value)
    template <typename F>
    __device__ __forceinline__ void each(F&& f) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) f(e / 2, j * 8 + 2 * t + e % 2, s[j][e]);
    }
    // f(row index, state of the tile, value, the other's value)
    template <typename F>
    __device__ __forceinline__ void each(Work& y, F&& f) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) f(e / 2, j * 8 + 2 * t + e % 2, s[j][e], y.s[j][e]);
    }
    static constexpr int LANES = 4;                                // neighbouring lanes that share a row
    __device__ __forceinline__ void scale_out(const double (&f)[NR]) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] *= f[e / 2];
    }
    __device__ __forceinline__ void hand_over(double*) {}          // the weights stay in their registers
    __device__ __forceinline__ void weigh(const double*, const double* V, int rest, int D) {
        const double* v = V + 2 * t * S::LDV + 2 * g;
#pragma unroll
        for (int k = 0; k < NT; ++k) {
            if (k * 8 >= rest) break;
            const double a[4] = {s[k][0], s[k][2], s[k][1], s[k][3]};
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) {
                if (j * 16 >= D) break;
                const double2 x = *reinterpret_cast<const double2*>(v + k * 8 * S::LDV + j * 16);
                const double2 y = *reinterpret_cast<const double2*>(v + (k * 8 + 1) * S::LDV + j * 16);
                const double b0[2] = {x.x, y.x}, b1[2] = {x.y, y.y};
                dmma_16x8x8(o[2 * j], a, b0);
                dmma_16x8x8(o[2 * j + 1], a, b1);
            }
        }
    }
    // f(row index, channel, value)
    template <typename F>
    __device__ __forceinline__ void each_out(F&& f) const {
#pragma unroll
        for (int j = 0; j < DP / 16; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) f(i, j * 16 + 4 * t + e, o[2 * j + e % 2][i * 2 + e / 2]);
    }
};

template <int DP, int BK_>
struct Work<float, DP, BK_> {
    using S = WideShape<float, DP, BK_>;
    static constexpr int NR = 8;
    float s[NR][4];
    Pair<float> o[NR][DP / 32];
    int ty, tx;
    __device__ __forceinline__ Work() : ty(threadIdx.x / 16), tx(threadIdx.x % 16) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int e = 0; e < DP / 32; ++e) o[i][e] = both(0.f);
    }
    __device__ __forceinline__ int row(int i) const { return ty * NR + i; }
    template <int LDY = S::LDK>
    __device__ __forceinline__ void scores(const float* Q, const float* K, int, int D) {
        Pair<float> acc[NR][4];
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = both(0.f);
        const float *q = Q + ty * NR * S::LDQ, *k = K + tx * LDY;
#pragma unroll 2
        for (int d = 0; d < DP; d += 4) {
            if (d >= D) break;
            float4 y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(k + 16 * j * LDY + d);
#pragma unroll
            for (int i = 0; i < NR; ++i) {
                const float4 x = *reinterpret_cast<const float4*>(q + i * S::LDQ + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    acc[i][j] = fma2(Pair<float>{x.x, x.y}, Pair<float>{y[j].x, y[j].y}, acc[i][j]);
                    acc[i][j] = fma2(Pair<float>{x.z, x.w}, Pair<float>{y[j].z, y[j].w}, acc[i][j]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = across(acc[i][j]);
    }
    template <typename F>
    __device__ __forceinline__ void each(F&& f) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) f(i, tx + 16 * j, s[i][j]);
    }
    template <typename F>
    __device__ __forceinline__ void each(Work& y, F&& f) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) f(i, tx + 16 * j, s[i][j], y.s[i][j]);
    }
    static constexpr int LANES = 16;
    __device__ __forceinline__ void scale_out(const float (&f)[NR]) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int e = 0; e < DP / 32; ++e) o[i][e] = mul2(o[i][e], both(f[i]));
    }
    __device__ __forceinline__ void hand_over(float* P) {
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) P[row(i) * S::LDP + tx + 16 * j] = s[i][j];
        __syncwarp();                      // a row's weights are read by the warp that wrote them
    }
    __device__ __forceinline__ void weigh(const float* P, const float* V, int rest, int) {
        const float *p = P + ty * NR * S::LDP, *v = V + tx * 4;
#pragma unroll 1
        for (int k = 0; k < S::BK && k < rest; k += 4) {
            float4 x[NR];
#pragma unroll
            for (int i = 0; i < NR; ++i) x[i] = *reinterpret_cast<const float4*>(p + i * S::LDP + k);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < DP / 64; ++c) {
                    const float4 y = *reinterpret_cast<const float4*>(v + (k + e) * S::LDV + 64 * c);
#pragma unroll
                    for (int i = 0; i < NR; ++i) {
                        const float w = e == 0 ? x[i].x : (e == 1 ? x[i].y : (e == 2 ? x[i].z : x[i].w));
                        o[i][2 * c] = fma2(both(w), Pair<float>{y.x, y.y}, o[i][2 * c]);
                        o[i][2 * c + 1] = fma2(both(w), Pair<float>{y.z, y.w}, o[i][2 * c + 1]);
                    }
                }
        }
    }
    template <typename F>
    __device__ __forceinline__ void each_out(F&& f) const {
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int c = 0; c < DP / 64; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) f(i, 64 * c + tx * 4 + e, e % 2 ? o[i][2 * c + e / 2].y : o[i][2 * c + e / 2].x);
    }
};

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 4 && DP == 64 ? 3 : 1)
attn_fwd_wide_kernel(AttnArgs a, bool vec) {
    using S = WideShape<T, DP>;
    using W = Work<T, DP>;
    constexpr int NR = W::NR;
    extern __shared__ __align__(128) unsigned char raw[];
    T* Qs = reinterpret_cast<T*>(raw);
    T *Ks = Qs + S::NQ, *Vs = Ks + S::NK, *Ps = Vs + S::NV;
    __shared__ T all_m[BQ], all_l[BQ];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), world = int(cluster.num_blocks());
    // rows: the positions of all query heads that share a state head, heads of a position side by side
    const int G = a.Hq / a.Hkv, rows = a.Lq * G;
    const int tiles = (rows + BQ - 1) / BQ;
    const int unit = int(blockIdx.x) / world;
    const int q0 = unit % tiles * BQ;
    const int g = unit / tiles % a.Hkv, b = unit / tiles / a.Hkv;
    const int n = attn_len(a, b);
    auto q_at = [&](int r) { return G == 1 ? r * a.qs[1] : int64_t(r / G) * a.qs[1] + int64_t(r % G) * a.qs[2]; };
    auto o_at = [&](int r) { return G == 1 ? r * a.os[1] : int64_t(r / G) * a.os[1] + int64_t(r % G) * a.os[2]; };
    auto k_at = [&](int r) { return int64_t(r) * a.ks[1]; };
    auto v_at = [&](int r) { return int64_t(r) * a.vs[1]; };
    auto lse_at = [&](int r) { return (int64_t(b) * a.Hq + g * G + r % G) * a.Lq + r / G; };
    const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + g * a.ks[2];
    const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + g * a.vs[2];
    const T c = T(a.scale * LOG2E), ninf = -INFINITY;
    const int steps = (n + S::BK - 1) / S::BK;
    W w;
    T m[NR], l[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) { m[i] = ninf; l[i] = 0; }
    if (rank < steps) {
        load_rows<T, BQ, DP, S::LDQ>(Qs, static_cast<const T*>(a.q) + b * a.qs[0] + int64_t(g) * G * a.qs[2], q_at, q0, rows, a.D, vec);
        load_rows<T, S::BK, DP, S::LDK>(Ks, k, k_at, rank * S::BK, n, a.D, vec);
    }
    for (int it = rank; it < steps; it += world) {
        const int k0 = it * S::BK;
        load_rows<T, S::BK, DP, S::LDV>(Vs, v, v_at, k0, n, a.D, vec);
        cp_async_wait<1>();
        __syncthreads();
        w.scores(Qs, Ks, n - k0, a.D);
        __syncthreads();
        if (it + world < steps) load_rows<T, S::BK, DP, S::LDK>(Ks, k, k_at, (it + world) * S::BK, n, a.D, vec);
        else cp_async_commit();
        T top[NR], f[NR], base[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i) top[i] = ninf;
        const int rest = n - k0;
        w.each([&](int i, int j, T& x) {
            x = j < rest ? x * c : ninf;
            top[i] = x > top[i] ? x : top[i];
        });
        bool moved = false;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
#pragma unroll
            for (int o = W::LANES / 2; o > 0; o >>= 1) {
                const T y = __shfl_xor_sync(0xffffffffu, top[i], o, 32);
                top[i] = y > top[i] ? y : top[i];
            }
            const T mn = top[i] > m[i] ? top[i] : m[i];
            base[i] = mn == ninf ? T(0) : mn;
            moved = moved || mn != m[i];
            f[i] = mn != m[i] ? exp_acc(m[i] - base[i]) : T(1);
            m[i] = mn;
            l[i] *= f[i];
        }
        if (__any_sync(0xffffffffu, moved)) w.scale_out(f);
        w.each([&](int i, int j, T& x) {
            x = j < rest ? exp_acc(x - base[i]) : T(0);
            l[i] += x;
        });
        w.hand_over(Ps);
        cp_async_wait<1>();
        __syncthreads();
        w.weigh(Ps, Vs, rest, a.D);
        __syncthreads();
    }
    cp_async_wait<0>();
#pragma unroll
    for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int o = W::LANES / 2; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o, 32);
    T* out = static_cast<T*>(const_cast<void*>(a.o)) + b * a.os[0] + int64_t(g) * G * a.os[2];
    const bool first = threadIdx.x % W::LANES == 0;
    if (world == 1) {
        T f[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            f[i] = n > 0 ? T(1) / l[i] : T(0);
            const int r = q0 + w.row(i);
            if (a.lse && first && r < rows)
                static_cast<T*>(a.lse)[lse_at(r)] = n > 0 ? m[i] / T(LOG2E) + log_acc(l[i]) : ninf;
        }
        T* to[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i) to[i] = q0 + w.row(i) < rows ? out + o_at(q0 + w.row(i)) : nullptr;
        w.each_out([&](int i, int d, T x) {
            if (to[i] && d < a.D) to[i][d] = x * f[i];
        });
        return;
    }
    // the blocks of a cluster: each leaves its rows over its tiles, then writes a share of the rows
    __syncthreads();
    T* mine = Qs;                                                  // [BQ][DP]
    static_assert(BQ * DP <= S::NQ, "");
    w.each_out([&](int i, int d, T x) { mine[w.row(i) * DP + d] = x; });
#pragma unroll
    for (int i = 0; i < NR; ++i)
        if (first) { all_m[w.row(i)] = m[i]; all_l[w.row(i)] = l[i]; }
    cluster.sync();
    for (int i = rank * THREADS + threadIdx.x; i < BQ * DP; i += world * THREADS) {
        const int r = i / DP, d = i % DP;
        if (q0 + r >= rows) continue;
        T top = ninf, sum = 0, x = 0;
        for (int p = 0; p < world; ++p) {
            const T y = *cluster.map_shared_rank(&all_m[r], p);
            top = y > top ? y : top;
        }
        const T base = top == ninf ? T(0) : top;
        for (int p = 0; p < world; ++p) {
            const T f = exp_acc(*cluster.map_shared_rank(&all_m[r], p) - base);
            sum += *cluster.map_shared_rank(&all_l[r], p) * f;
            x += *cluster.map_shared_rank(&mine[i], p) * f;
        }
        if (d < a.D) out[o_at(q0 + r) + d] = n > 0 ? x / sum : T(0);
        if (d == 0 && a.lse) static_cast<T*>(a.lse)[lse_at(q0 + r)] = n > 0 ? top / T(LOG2E) + log_acc(sum) : ninf;
    }
    cluster.sync();                        // nobody leaves while its shared memory is read
}

// ---------------------------------------------------------------------------
// Backward, with the roles of the tensor-core kernels: a block keeps 64 rows (positions for dQ, states for dK and dV), streams
// tiles of the other side, and sums its rows' gradients in registers in a fixed order.  Streamed tiles are the second
// operand of the scores and of the gradients, so their row stride suits both.

template <typename T, int DP>
struct BwdWide {
    static constexpr bool F64 = sizeof(T) == 8;
    static constexpr int BK = F64 ? (DP == 128 ? 16 : 32) : 64;
    using S = WideShape<T, DP, BK>;
    static constexpr int NA = BQ * S::LDQ, NB = BK * S::LDV;
    static constexpr int BYTES = (2 * NA + 2 * NB + S::NP + 2 * BK) * int(sizeof(T));
    // dK and dV of 128 channels in double do not fit the registers together: one pass each
    static constexpr bool APART = F64 && DP == 128;
};

constexpr int BOTH = 0, ONLY_V = 1, ONLY_K = 2;

template <typename T, int DP, bool KV, int WHICH>
__global__ void __launch_bounds__(THREADS)
attn_bwd_wide_kernel(AttnArgs a, bool vec) {
    using H = BwdWide<T, DP>;
    using S = typename H::S;
    using W = Work<T, DP, H::BK>;
    constexpr int NR = W::NR, BK = H::BK;
    extern __shared__ __align__(128) unsigned char raw[];
    T* A0 = reinterpret_cast<T*>(raw);
    T *A1 = A0 + H::NA, *B0 = A1 + H::NA, *B1 = B0 + H::NB, *Ps = B1 + H::NB, *col_l = Ps + S::NP, *col_d = col_l + BK;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), world = int(cluster.num_blocks());
    const int G = a.Hq / a.Hkv, rows = a.Lq * G;
    const int own = KV ? a.Lk : rows;
    const int tiles = (own + BQ - 1) / BQ;
    const int unit = int(blockIdx.x) / world;
    const int r0 = unit % tiles * BQ;
    const int g = unit / tiles % a.Hkv, b = unit / tiles / a.Hkv;
    const int n = attn_len(a, b);
    const int own_n = KV ? n : rows, other_n = KV ? rows : n;
    const int steps = r0 < own_n ? (other_n + BK - 1) / BK : 0;
    auto at = [&](const int64_t (&s)[3], int r) { return G == 1 ? r * s[1] : int64_t(r / G) * s[1] + int64_t(r % G) * s[2]; };
    auto q_at = [&](int r) { return at(a.qs, r); };
    auto g_at = [&](int r) { return at(a.dos, r); };
    auto k_at = [&](int r) { return int64_t(r) * a.ks[1]; };
    auto v_at = [&](int r) { return int64_t(r) * a.vs[1]; };
    auto stat_at = [&](int r) {
        return G == 1 ? (int64_t(b) * a.Hq + g) * a.Lq + r : (int64_t(b) * a.Hq + g * G + r % G) * a.Lq + r / G;
    };
    const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + int64_t(g) * G * a.qs[2];
    const T* go = static_cast<const T*>(a.dout) + b * a.dos[0] + int64_t(g) * G * a.dos[2];
    const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + g * a.ks[2];
    const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + g * a.vs[2];
    const T *lse = static_cast<const T*>(a.lse), *delta = static_cast<const T*>(a.delta);
    const T c = T(a.scale * LOG2E);
    auto load0 = [&](int it) {
        if (it >= steps) { cp_async_commit(); return; }
        if constexpr (KV) load_rows<T, BK, DP, S::LDV>(B0, q, q_at, it * BK, rows, a.D, vec);
        else load_rows<T, BK, DP, S::LDV>(B0, k, k_at, it * BK, n, a.D, vec);
    };
    auto load1 = [&](int it) {
        if (it >= steps) { cp_async_commit(); return; }
        if constexpr (KV) load_rows<T, BK, DP, S::LDV>(B1, go, g_at, it * BK, rows, a.D, vec);
        else load_rows<T, BK, DP, S::LDV>(B1, v, v_at, it * BK, n, a.D, vec);
    };
    const bool busy = r0 + int(threadIdx.x / 32) * 16 < own_n;    // a warp has 16 rows
    W x, y;                                // S (then P) with dV; dP (then dS) with dK or dQ
    T row_l[NR], row_d[NR];
    if (rank < steps) {
        if constexpr (KV) {
            load_rows<T, BQ, DP, S::LDQ>(A0, k, k_at, r0, n, a.D, vec);
            load_rows<T, BQ, DP, S::LDQ>(A1, v, v_at, r0, n, a.D, vec);
        } else {
            load_rows<T, BQ, DP, S::LDQ>(A0, q, q_at, r0, rows, a.D, vec);
            load_rows<T, BQ, DP, S::LDQ>(A1, go, g_at, r0, rows, a.D, vec);
        }
        load0(rank);
        load1(rank);
    }
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int r = r0 + x.row(i);
        row_l[i] = !KV && r < rows ? lse[stat_at(r)] * T(LOG2E) : T(0);
        row_d[i] = !KV && r < rows ? delta[stat_at(r)] : T(0);
    }
    for (int it = rank; it < steps; it += world) {
        const int rest = other_n - it * BK;
        if (KV)
            for (int j = threadIdx.x; j < BK && j < rest; j += THREADS) {
                col_l[j] = lse[stat_at(it * BK + j)] * T(LOG2E);
                col_d[j] = delta[stat_at(it * BK + j)];
            }
        cp_async_wait<0>();
        __syncthreads();
        if (busy) x.template scores<S::LDV>(A0, B0, rest, a.D);
        if (WHICH != ONLY_V && busy) y.template scores<S::LDV>(A1, B1, rest, a.D);
        if (!KV) {
            __syncthreads();
            load1(it + world);
        }
        if (busy) x.each(y, [&](int i, int j, T& p, T& d) {
            const T l = KV ? (j < rest ? col_l[j] : T(0)) : row_l[i];
            p = j < rest ? exp_acc(p * c - l) : T(0);
            if (WHICH != ONLY_V) d = j < rest ? p * (d - (KV ? col_d[j] : row_d[i])) : T(0);
        });
        if (KV && WHICH != ONLY_K && busy) {
            x.hand_over(Ps);
            x.weigh(Ps, B1, rest, a.D);
        }
        if (KV) {
            __syncthreads();
            load1(it + world);
        }
        if (WHICH != ONLY_V && busy) {
            y.hand_over(Ps);
            y.weigh(Ps, B0, rest, a.D);
        }
        __syncthreads();
        load0(it + world);
    }
    cp_async_wait<0>();
    auto dense_at = [&](int r) {
        return KV ? ((int64_t(b) * a.Lk + r) * a.Hkv + g) * a.D
                  : (G == 1 ? ((int64_t(b) * a.Lq + r) * a.Hq + g) * a.D : ((int64_t(b) * a.Lq + r / G) * a.Hq + g * G + r % G) * a.D);
    };
    T *out_y = static_cast<T*>(KV ? a.dk : a.dq), *out_x = static_cast<T*>(a.dv);
    if (world == 1) {
        int64_t to[NR];
#pragma unroll
        for (int i = 0; i < NR; ++i) to[i] = r0 + x.row(i) < own ? dense_at(r0 + x.row(i)) : -1;
        if (WHICH != ONLY_V)
            y.each_out([&](int i, int d, T z) {
                if (to[i] >= 0 && d < a.D) out_y[to[i] + d] = r0 + x.row(i) < own_n ? z * T(a.scale) : T(0);
            });
        if (KV && WHICH != ONLY_K)
            x.each_out([&](int i, int d, T z) {
                if (to[i] >= 0 && d < a.D) out_x[to[i] + d] = r0 + x.row(i) < own_n ? z : T(0);
            });
        return;
    }
    __syncthreads();
    static_assert(BQ * DP <= H::NA, "");
    if (WHICH != ONLY_V) y.each_out([&](int i, int d, T z) { A0[x.row(i) * DP + d] = z; });
    if (KV && WHICH != ONLY_K) x.each_out([&](int i, int d, T z) { A1[x.row(i) * DP + d] = z; });
    cluster.sync();
    for (int i = rank * THREADS + threadIdx.x; i < BQ * DP; i += world * THREADS) {
        const int r = r0 + i / DP, d = i % DP;
        if (r >= own || d >= a.D) continue;
        T sum_y = 0, sum_x = 0;
        for (int w = 0; w < world; ++w) {
            if (WHICH != ONLY_V) sum_y += *cluster.map_shared_rank(A0 + i, w);
            if (KV && WHICH != ONLY_K) sum_x += *cluster.map_shared_rank(A1 + i, w);
        }
        const bool in = r < own_n;
        if (WHICH != ONLY_V) out_y[dense_at(r) + d] = in ? sum_y * T(a.scale) : T(0);
        if (KV && WHICH != ONLY_K) out_x[dense_at(r) + d] = in ? sum_x : T(0);
    }
    cluster.sync();                        // nobody leaves while its shared memory is read
}

// 16-byte accesses on every row?
bool wide_rows16(const AttnArgs& a, int64_t e, bool backward) {
    bool vec = a.D * e % 16 == 0;
    for (auto* s : {a.qs, a.ks, a.vs, backward ? a.dos : a.qs})
        for (int i = 0; i < 3; ++i) vec = vec && s[i] * e % 16 == 0;
    for (const void* p : {a.q, a.k, a.v, backward ? a.dout : a.q}) vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    return vec;
}

// `units` blocks, or clusters of up to 16 where blocks are few: those share the `steps` tiles a block walks over, two each at least
template <typename K>
int launch_wide(K kernel, int64_t units, int64_t steps, int per_sm, int smem, cudaStream_t st, const AttnArgs& a, bool vec) {
    const int sms = sm_count();
    int world = 1;
    while (world < 16 && units * world * 2 <= int64_t(sms) * per_sm && world * 4 <= steps) world *= 2;
    // or where the last blocks would leave many SMs idle: the longest sum of an SM's blocks counts
    auto longest = [&](int w) { return double(ceil_div(units * w, sms)) / w; };
    for (int w = 2; world == 1 && w <= 4 && w * 4 <= steps; w *= 2)
        if (longest(w) < 0.9 * longest(1)) world = w;
    NNVB_REQUIRE(units * world < (int64_t(1) << 31), "nnvb_cross_attention: too many tiles (%lld) for one launch", (long long)units);
    NNVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (world > 8) NNVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(units * world));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = size_t(smem);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = unsigned(world);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    NNVB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, vec));
    return NNVB_OK;
}

template <typename T, int DP>
int wide_backward_t(cudaStream_t st, const AttnArgs& a) {
    using H = BwdWide<T, DP>;
    const bool vec = wide_rows16(a, sizeof(T), true);
    const int64_t rows = int64_t(a.Lq) * (a.Hq / a.Hkv), heads = int64_t(a.Hkv) * a.B;
    const int per_sm = H::BYTES <= 113 * 1024 ? 2 : 1;
    const int64_t uk = ceil_div(a.Lk, BQ) * heads, sk = ceil_div(rows, H::BK);
    NNVB_TRY(launch_wide(attn_bwd_wide_kernel<T, DP, false, BOTH>, ceil_div(rows, BQ) * heads, ceil_div(a.Lk, H::BK), per_sm,
                         H::BYTES, st, a, vec));
    if constexpr (H::APART) {
        NNVB_TRY(launch_wide(attn_bwd_wide_kernel<T, DP, true, ONLY_V>, uk, sk, per_sm, H::BYTES, st, a, vec));
        return launch_wide(attn_bwd_wide_kernel<T, DP, true, ONLY_K>, uk, sk, per_sm, H::BYTES, st, a, vec);
    } else {
        return launch_wide(attn_bwd_wide_kernel<T, DP, true, BOTH>, uk, sk, per_sm, H::BYTES, st, a, vec);
    }
}

template <typename T, int DP>
int wide_t(cudaStream_t st, const AttnArgs& a) {
    using S = WideShape<T, DP>;
    const bool vec = wide_rows16(a, sizeof(T), false);
    return launch_wide(attn_fwd_wide_kernel<T, DP>, ceil_div(int64_t(a.Lq) * (a.Hq / a.Hkv), BQ) * a.Hkv * a.B,
                       ceil_div(a.Lk, S::BK), 2, S::BYTES, st, a, vec);
}

}  // namespace

int attn_forward_wide(cudaStream_t st, const AttnArgs& a) {
    if (a.dtype == NNVB_F64) return a.D <= 64 ? wide_t<double, 64>(st, a) : wide_t<double, 128>(st, a);
    return a.D <= 64 ? wide_t<float, 64>(st, a) : wide_t<float, 128>(st, a);
}

int attn_backward_wide(cudaStream_t st, const AttnArgs& a) {
    if (a.dtype == NNVB_F64) return a.D <= 64 ? wide_backward_t<double, 64>(st, a) : wide_backward_t<double, 128>(st, a);
    return a.D <= 64 ? wide_backward_t<float, 64>(st, a) : wide_backward_t<float, 128>(st, a);
}

}  // namespace nnvb
