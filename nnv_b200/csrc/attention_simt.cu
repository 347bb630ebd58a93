// Attention over an encoder's states on the CUDA cores: the layouts the tensor-core kernels do not
// take (16-bit rows that are not 16-byte aligned, heads of more than 128 channels in any type), and the backward pass
// of small or one-sided problems in float and double.
//
//   forward   one pass over the states with the running maximum m and sum l of each row's softmax:
//             m' = max(m, max_j S_j), p_j = exp(S_j - m'), l' = l exp(m - m') + sum p_j, O' = O exp(m - m') + p V
//   backward  P = exp(S - lse), dP = dO V^T, dS = P (dP - delta), delta = sum_d dO O;  dQ = scale dS K (a block per
//             tile of positions, walking over the states), dK = scale dS^T Q and dV = P^T dO (a block per tile of
//             states, walking over the positions of every query head that shares it): nothing is added atomically
//
// A block of 256 threads holds TILE x TILE scores, 16 x 16 threads with (TILE/16)^2 scores each, operands in shared
// memory in the type sums are held in, rows padded by 16 bytes so that the 16-byte loads of neighbouring rows
// fall on different banks.  With 64 rows a 4 x 4 register tile needs 8 16-byte loads for 64 FMAs.
// Problems with a short side are bound by the latency of a step (load, products, exponentials, products; a short side also
// leaves warps of the products over it idle), so two blocks share an SM: 18 x 1618 x 8 x 2 x 2 x 128 float 392 us, 2 x 3178 x
// 19 x 2 x 4 x 96 double 681 us.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "attention.cuh"
#include "mma_f64.cuh"

namespace cg = cooperative_groups;

namespace nnvb {
namespace {

constexpr int THREADS = 256;

// Rows are the positions of all query heads that share a state head, heads of a position side by side, so that few
// positions of grouped heads fill tiles.
struct Rows {
    int G, n;                                      // heads of the group, rows
    const AttnArgs& a;
    int b, g;
    __device__ Rows(const AttnArgs& a_, int b_, int g_) : G(a_.Hq / a_.Hkv), n(a_.Lq * (a_.Hq / a_.Hkv)), a(a_), b(b_), g(g_) {}
    // of a tensor with strides s, from the group's first head
    __device__ __forceinline__ int64_t at(const int64_t (&s)[3], int r) const {
        return G == 1 ? r * s[1] : int64_t(r / G) * s[1] + int64_t(r % G) * s[2];
    }
    __device__ __forceinline__ int64_t first(const int64_t (&s)[3]) const { return int64_t(b) * s[0] + int64_t(g) * G * s[2]; }
    // of a [B, Hq, Lq] statistic; of the dense gradient of q
    __device__ __forceinline__ int64_t stat(int r) const {
        return G == 1 ? (int64_t(b) * a.Hq + g) * a.Lq + r : (int64_t(b) * a.Hq + g * G + r % G) * a.Lq + r / G;
    }
    __device__ __forceinline__ int64_t dense(int r) const {
        return G == 1 ? ((int64_t(b) * a.Lq + r) * a.Hq + g) * a.D : ((int64_t(b) * a.Lq + r / G) * a.Hq + g * G + r % G) * a.D;
    }
};

template <typename A> struct VecOf;
template <> struct VecOf<float> { static constexpr int N = 4; };
template <> struct VecOf<double> { static constexpr int N = 2; };

template <typename A>
__device__ __forceinline__ Pack<A, VecOf<A>::N> lds(const A* p) {
    return *reinterpret_cast<const Pack<A, VecOf<A>::N>*>(p);
}

// rows [r0, r0 + TILE) into s[TILE][DP + pad]; row r begins at(r) elements from g; rows at or past n_rows and columns past
// D are zero.  vec: rows of float and double arrive asynchronously
template <typename T, typename A, int TILE, int DP, typename At>
__device__ void load_tile(A* s, const T* g, At&& at, int r0, int n_rows, int D, bool vec) {
    constexpr int LD = DP + VecOf<A>::N;
    constexpr int V = 16 / sizeof(T);
    if (vec && std::is_same<T, A>::value) {
#pragma unroll 4
        for (int i = threadIdx.x; i < TILE * (DP / V); i += THREADS) {
            const int r = i / (DP / V), c = i % (DP / V) * V;
            const bool in = r0 + r < n_rows && c < D;
            cp_async16(s + r * LD + c, g + (in ? at(r0 + r) + c : 0), in ? 16 : 0);
        }
        cp_async_commit();
    } else if (vec) {
#pragma unroll 4
        for (int i = threadIdx.x; i < TILE * (DP / V); i += THREADS) {
            const int r = i / (DP / V), c = i % (DP / V) * V;
            Pack<T, V> p;
            const bool in = r0 + r < n_rows && c < D;          // D is a multiple of V here
            if (in) p = *reinterpret_cast<const Pack<T, V>*>(g + at(r0 + r) + c);
#pragma unroll
            for (int e = 0; e < V; ++e) s[r * LD + c + e] = in ? to_acc(p.v[e]) : A(0);
        }
    } else {
        for (int i = threadIdx.x; i < TILE * DP; i += THREADS) {
            const int r = i / DP, c = i % DP;
            s[r * LD + c] = r0 + r < n_rows && c < D ? A(to_acc(g[at(r0 + r) + c])) : A(0);
        }
    }
}

// acc[i][j] += sum_d X[(ty*M + i)][d] * Y[tx + 16 j][d], d < D; rows of X from nx on and of Y from ny on do not count
template <typename A, int TILE, int DP>
__device__ __forceinline__ void mul_rows(A (&acc)[TILE / 16][TILE / 16], const A* X, const A* Y, int D, int nx, int ny, int ty, int tx) {
    constexpr int M = TILE / 16, V = VecOf<A>::N, LD = DP + V;
    if (int(threadIdx.x / 32) * 2 * M >= nx) return;       // none of this warp's rows
    auto step = [&](int d) {
        Pack<A, V> x[M], y[M];
#pragma unroll
        for (int i = 0; i < M; ++i) x[i] = lds<A>(X + (ty * M + i) * LD + d);
#pragma unroll
        for (int j = 0; j < M; ++j)
            if (16 * j < ny) {
                y[j] = lds<A>(Y + (tx + 16 * j) * LD + d);
#pragma unroll
                for (int e = 0; e < V; ++e)
#pragma unroll
                    for (int i = 0; i < M; ++i) acc[i][j] += x[i].v[e] * y[j].v[e];
            }
    };
    if (D > DP - V) {                      // a loop of known length is the faster one
#pragma unroll 4
        for (int d = 0; d < DP; d += V) step(d);
    } else {
#pragma unroll 2
        for (int d = 0; d < D; d += V) step(d);
    }
}

// acc[i][c] += sum_k P[ty*M + i][k] * Y[k][column c of this thread], k < n;  thread columns: V at tx*V + 16*V*c
template <typename A, int TILE, int DP>
__device__ __forceinline__ void mul_cols(A (&acc)[TILE / 16][DP / 16], const A* P, const A* Y, int n, int ty, int tx) {
    constexpr int M = TILE / 16, V = VecOf<A>::N, LD = DP + V, LP = TILE + V, NC = DP / (16 * V);
#pragma unroll 2
    for (int k = 0; k < TILE && k < n; k += V) {
        Pack<A, V> p[M];
#pragma unroll
        for (int i = 0; i < M; ++i) p[i] = lds<A>(P + (ty * M + i) * LP + k);
#pragma unroll
        for (int e = 0; e < V; ++e)
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const Pack<A, V> y = lds<A>(Y + (k + e) * LD + tx * V + 16 * V * c);
#pragma unroll
                for (int i = 0; i < M; ++i)
#pragma unroll
                    for (int f = 0; f < V; ++f) acc[i][c * V + f] += p[i].v[e] * y.v[f];
            }
    }
}

// acc[i][c] += sum_q P[q][ty*M + i] * Y[q][column c of this thread], q < n; rows of the result from nr on do not count
template <typename A, int TILE, int DP>
__device__ __forceinline__ void mul_cols_t(A (&acc)[TILE / 16][DP / 16], const A* P, const A* Y, int n, int nr, int ty, int tx) {
    constexpr int M = TILE / 16, V = VecOf<A>::N, LD = DP + V, LP = TILE + V, NC = DP / (16 * V);
    if (int(threadIdx.x / 32) * 2 * M >= nr) return;       // none of this warp's rows
#pragma unroll 4
    for (int q = 0; q < TILE && q < n; ++q) {
        A p[M];
#pragma unroll
        for (int i = 0; i < M; ++i) p[i] = P[q * LP + ty * M + i];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const Pack<A, V> y = lds<A>(Y + q * LD + tx * V + 16 * V * c);
#pragma unroll
            for (int i = 0; i < M; ++i)
#pragma unroll
                for (int f = 0; f < V; ++f) acc[i][c * V + f] += p[i] * y.v[f];
        }
    }
}

template <typename T, typename A, int TILE, int DP, typename At>
__device__ __forceinline__ void store_rows(T* g, At&& at, int r0, int n_rows, int D, const A (&acc)[TILE / 16][DP / 16],
                                           const A (&f)[TILE / 16], int ty, int tx) {
    constexpr int M = TILE / 16, V = VecOf<A>::N, NC = DP / (16 * V);
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const int r = r0 + ty * M + i;
        T* to = g + (r < n_rows ? at(r) : 0);
        if (r < n_rows)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const int d = tx * V + 16 * V * c + e;
                    if (d < D) to[d] = from_acc<T, A>(acc[i][c * V + e] * f[i]);
                }
    }
}

// The blocks of a cluster have summed shares of the same rows: each leaves its sums in `mine`, [TILE][DP], and writes a
// share of the total, added in block order.
template <typename T, typename A, int TILE, int DP, typename At>
__device__ void store_shared(cg::cluster_group& cluster, T* g, At&& at, int r0, int n_rows, int D, const A* mine, A f) {
    const int rank = int(cluster.block_rank()), world = int(cluster.num_blocks());
    for (int i = rank * THREADS + threadIdx.x; i < TILE * DP; i += world * THREADS) {
        const int r = r0 + i / DP, d = i % DP;
        if (r >= n_rows || d >= D) continue;
        A x = 0;
        for (int p = 0; p < world; ++p) x += *cluster.map_shared_rank(mine + i, p);
        g[at(r) + d] = from_acc<T, A>(x * f);
    }
}
template <typename A, int TILE, int DP>
__device__ void leave_rows(A* mine, const A (&acc)[TILE / 16][DP / 16], int ty, int tx) {
    constexpr int M = TILE / 16, V = VecOf<A>::N, NC = DP / (16 * V);
#pragma unroll
    for (int i = 0; i < M; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) mine[(ty * M + i) * DP + tx * V + 16 * V * c + e] = acc[i][c * V + e];
}

template <typename A>
__device__ __forceinline__ A max16(A x) {
    for (int o = 8; o > 0; o >>= 1) {
        const A y = __shfl_xor_sync(0xffffffffu, x, o, 32);
        x = y > x ? y : x;
    }
    return x;
}
template <typename A>
__device__ __forceinline__ A sum16(A x) {
    for (int o = 8; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o, 32);
    return x;
}

template <typename T, int TILE, int DP>
__global__ void __launch_bounds__(THREADS)
attn_fwd_simt_kernel(AttnArgs a, bool vec) {
    using A = typename AccOf<T>::type;
    constexpr int M = TILE / 16, V = VecOf<A>::N, LD = DP + V, LP = TILE + V;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    A* Qs = reinterpret_cast<A*>(smem_raw);
    A* Ks = Qs + TILE * LD;
    A* Vs = Ks + TILE * LD;
    A* Ps = Vs + TILE * LD;
    const int tiles = (a.Lq * (a.Hq / a.Hkv) + TILE - 1) / TILE;
    const int q0 = int(blockIdx.x % tiles) * TILE;
    const int g = int(blockIdx.x / tiles % a.Hkv), b = int(blockIdx.x / tiles / a.Hkv);
    const Rows rows(a, b, g);
    const int n = attn_len(a, b);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const T* q = static_cast<const T*>(a.q) + rows.first(a.qs);
    const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + g * a.ks[2];
    const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + g * a.vs[2];
    const A c = A(a.scale * LOG2E), ninf = -INFINITY;
    A o[M][DP / 16], m[M], l[M];
#pragma unroll
    for (int i = 0; i < M; ++i) {
        m[i] = ninf;
        l[i] = 0;
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) o[i][e] = 0;
    }
    load_tile<T, A, TILE, DP>(Qs, q, [&](int r) { return rows.at(a.qs, r); }, q0, rows.n, a.D, vec);
    for (int k0 = 0; k0 < n; k0 += TILE) {
        __syncthreads();
        load_tile<T, A, TILE, DP>(Ks, k, [&](int r) { return r * a.ks[1]; }, k0, n, a.D, vec);
        load_tile<T, A, TILE, DP>(Vs, v, [&](int r) { return r * a.vs[1]; }, k0, n, a.D, vec);
        cp_async_wait<0>();
        __syncthreads();
        A s[M][M] = {};
        mul_rows<A, TILE, DP>(s, Qs, Ks, a.D, rows.n - q0, n - k0, ty, tx);
#pragma unroll
        for (int i = 0; i < M; ++i) {
            A mx = ninf;
#pragma unroll
            for (int j = 0; j < M; ++j) {
                s[i][j] = k0 + tx + 16 * j < n ? s[i][j] * c : ninf;
                mx = s[i][j] > mx ? s[i][j] : mx;
            }
            mx = max16(mx);
            const A mn = mx > m[i] ? mx : m[i];
            const A base = mn == ninf ? A(0) : mn;       // every score so far is -inf: exp(-inf - 0) = 0
            const A f = exp_acc(m[i] - base);
            m[i] = mn;
            A t = 0;
#pragma unroll
            for (int j = 0; j < M; ++j) {
                const A p = exp_acc(s[i][j] - base);
                t += p;
                Ps[(ty * M + i) * LP + tx + 16 * j] = p;
            }
            l[i] = l[i] * f + sum16(t);
#pragma unroll
            for (int e = 0; e < DP / 16; ++e) o[i][e] *= f;
        }
        __syncwarp();                     // a warp reads back only the rows its own threads wrote
        mul_cols<A, TILE, DP>(o, Ps, Vs, n - k0, ty, tx);
    }
    cp_async_wait<0>();
    A f[M];
#pragma unroll
    for (int i = 0; i < M; ++i) {
        f[i] = n > 0 ? A(1) / l[i] : A(0);
        const int r = q0 + ty * M + i;
        if (a.lse && tx == 0 && r < rows.n)
            static_cast<A*>(a.lse)[rows.stat(r)] = n > 0 ? m[i] / A(LOG2E) + log_acc(l[i]) : ninf;
    }
    T* out = static_cast<T*>(const_cast<void*>(a.o)) + rows.first(a.os);
    store_rows<T, A, TILE, DP>(out, [&](int r) { return rows.at(a.os, r); }, q0, rows.n, a.D, o, f, ty, tx);
}

template <typename T>
__global__ void __launch_bounds__(256)
attn_delta_kernel(AttnArgs a) {
    using A = typename AccOf<T>::type;
    const int lane = threadIdx.x % 32;
    const int64_t i = int64_t(blockIdx.x) * 8 + threadIdx.x / 32;      // ((b * Lq) + r) * Hq + h
    if (i >= int64_t(a.B) * a.Lq * a.Hq) return;
    const int h = int(i % a.Hq), r = int(i / a.Hq % a.Lq), b = int(i / a.Hq / a.Lq);
    const T* o = static_cast<const T*>(a.o) + b * a.os[0] + r * a.os[1] + h * a.os[2];
    const T* d = static_cast<const T*>(a.dout) + b * a.dos[0] + r * a.dos[1] + h * a.dos[2];
    A s = 0;
    for (int c = lane; c < a.D; c += 32) s += A(to_acc(o[c])) * A(to_acc(d[c]));
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w, 32);
    if (lane == 0) static_cast<A*>(a.delta)[(int64_t(b) * a.Hq + h) * a.Lq + r] = s;
}

// dQ: a block per tile of positions.  16-bit types: delta comes from a rounded output (delta0), and where a row's weight lies
// on a few states that rounding is larger than dP - delta; so the sum e of P (dP - delta0) is taken back as dQ - e sum P K,
// and delta0 + e is left for dK (4 x 512 x 512 x 8 x 256 bf16, both passes: 2.27 ms without, 2.44 with).
template <typename T, int TILE, int DP>
__global__ void __launch_bounds__(THREADS)
attn_dq_simt_kernel(AttnArgs a, bool vec) {
    using A = typename AccOf<T>::type;
    constexpr int M = TILE / 16, V = VecOf<A>::N, LD = DP + V, LP = TILE + V;
    constexpr bool ROUNDED = sizeof(T) == 2;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    A* Qs = reinterpret_cast<A*>(smem_raw);
    A* Gs = Qs + TILE * LD;
    A* Ks = Gs + TILE * LD;
    A* Vs = Ks + TILE * LD;
    A* Ps = Vs + TILE * LD;
    A* Ws = Ps + TILE * LP;
    __shared__ A sums[TILE];
    const int tiles = (a.Lq * (a.Hq / a.Hkv) + TILE - 1) / TILE;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), world = int(cluster.num_blocks());
    const int unit = int(blockIdx.x) / world;
    const int q0 = unit % tiles * TILE;
    const int g = unit / tiles % a.Hkv, b = unit / tiles / a.Hkv;
    const Rows rows(a, b, g);
    const int n = attn_len(a, b);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + g * a.ks[2];
    const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + g * a.vs[2];
    A* delta = static_cast<A*>(a.delta);
    const A c = A(a.scale * LOG2E);
    A acc[M][DP / 16], w[M][ROUNDED ? DP / 16 : 1], lse[M], dl[M], f[M], miss[M];
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const int r = q0 + ty * M + i;
        lse[i] = r < rows.n ? static_cast<const A*>(a.lse)[rows.stat(r)] * A(LOG2E) : A(0);
        dl[i] = r < rows.n ? delta[rows.stat(r)] : A(0);
        f[i] = A(a.scale);
        miss[i] = 0;
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) {
            acc[i][e] = 0;
            if constexpr (ROUNDED) w[i][e] = 0;
        }
    }
    load_tile<T, A, TILE, DP>(Qs, static_cast<const T*>(a.q) + rows.first(a.qs), [&](int r) { return rows.at(a.qs, r); }, q0, rows.n, a.D, vec);
    load_tile<T, A, TILE, DP>(Gs, static_cast<const T*>(a.dout) + rows.first(a.dos), [&](int r) { return rows.at(a.dos, r); }, q0, rows.n, a.D, vec);
    for (int k0 = rank * TILE; k0 < n; k0 += world * TILE) {
        __syncthreads();
        load_tile<T, A, TILE, DP>(Ks, k, [&](int r) { return r * a.ks[1]; }, k0, n, a.D, vec);
        load_tile<T, A, TILE, DP>(Vs, v, [&](int r) { return r * a.vs[1]; }, k0, n, a.D, vec);
        cp_async_wait<0>();
        __syncthreads();
        A s[M][M] = {}, dp[M][M] = {};
        mul_rows<A, TILE, DP>(s, Qs, Ks, a.D, rows.n - q0, n - k0, ty, tx);
        mul_rows<A, TILE, DP>(dp, Gs, Vs, a.D, rows.n - q0, n - k0, ty, tx);
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
            for (int j = 0; j < M; ++j) {
                const A p = k0 + tx + 16 * j < n ? exp_acc(s[i][j] * c - lse[i]) : A(0), ds = p * (dp[i][j] - dl[i]);
                Ps[(ty * M + i) * LP + tx + 16 * j] = ds;
                if constexpr (ROUNDED) {
                    Ws[(ty * M + i) * LP + tx + 16 * j] = p;
                    miss[i] += ds;
                }
            }
        __syncwarp();
        mul_cols<A, TILE, DP>(acc, Ps, Ks, n - k0, ty, tx);
        if constexpr (ROUNDED) mul_cols<A, TILE, DP>(w, Ws, Ks, n - k0, ty, tx);
    }
    cp_async_wait<0>();
    if constexpr (ROUNDED)
#pragma unroll
        for (int i = 0; i < M; ++i) miss[i] = sum16(miss[i]);
    T* dq = static_cast<T*>(a.dq);
    auto at = [&](int r) { return rows.dense(r); };
    if (world == 1) {
        if constexpr (ROUNDED)
#pragma unroll
            for (int i = 0; i < M; ++i) {
#pragma unroll
                for (int e = 0; e < DP / 16; ++e) acc[i][e] -= miss[i] * w[i][e];
                const int r = q0 + ty * M + i;
                if (tx == 0 && r < rows.n) delta[rows.stat(r)] = dl[i] + miss[i];
            }
        store_rows<T, A, TILE, DP>(dq, at, q0, rows.n, a.D, acc, f, ty, tx);
        return;
    }
    __syncthreads();
    leave_rows<A, TILE, DP>(Qs, acc, ty, tx);
    if constexpr (ROUNDED) {
        leave_rows<A, TILE, DP>(Gs, w, ty, tx);
#pragma unroll
        for (int i = 0; i < M; ++i)
            if (tx == 0) sums[ty * M + i] = miss[i];
    }
    cluster.sync();
    if constexpr (ROUNDED) {
        for (int i = rank * THREADS + threadIdx.x; i < TILE * DP; i += world * THREADS) {
            const int r = q0 + i / DP, d = i % DP;
            if (r >= rows.n || d >= a.D) continue;
            A x = 0, y = 0, e = 0;
            for (int p = 0; p < world; ++p) {
                x += *cluster.map_shared_rank(Qs + i, p);
                y += *cluster.map_shared_rank(Gs + i, p);
                e += *cluster.map_shared_rank(sums + i / DP, p);
            }
            dq[at(r) + d] = from_acc<T, A>((x - e * y) * A(a.scale));
            if (d == 0) delta[rows.stat(r)] += e;
        }
    } else {
        store_shared<T, A, TILE, DP>(cluster, dq, at, q0, rows.n, a.D, Qs, A(a.scale));
    }
    cluster.sync();                        // nobody leaves while its shared memory is read
}

// dK, dV: a block per tile of states, over the positions of every query head of its group
template <typename T, int TILE, int DP>
__global__ void __launch_bounds__(THREADS)
attn_dkv_simt_kernel(AttnArgs a, bool vec) {
    using A = typename AccOf<T>::type;
    constexpr int M = TILE / 16, V = VecOf<A>::N, LD = DP + V, LP = TILE + V;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    A* Ks = reinterpret_cast<A*>(smem_raw);
    A* Vs = Ks + TILE * LD;
    A* Qs = Vs + TILE * LD;
    A* Gs = Qs + TILE * LD;
    A* Ps = Gs + TILE * LD;
    A* Ss = Ps + TILE * LP;
    const int tiles = (a.Lk + TILE - 1) / TILE;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), world = int(cluster.num_blocks());
    const int unit = int(blockIdx.x) / world;
    const int k0 = unit % tiles * TILE;
    const int g = unit / tiles % a.Hkv, b = unit / tiles / a.Hkv;
    const Rows rows(a, b, g);
    const int n = attn_len(a, b);
    const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
    const A c = A(a.scale * LOG2E);
    A dk[M][DP / 16], dv[M][DP / 16], fk[M], fv[M];
#pragma unroll
    for (int i = 0; i < M; ++i) {
        fk[i] = A(a.scale);
        fv[i] = 1;
#pragma unroll
        for (int e = 0; e < DP / 16; ++e) { dk[i][e] = 0; dv[i][e] = 0; }
    }
    if (k0 < n) {
        load_tile<T, A, TILE, DP>(Ks, static_cast<const T*>(a.k) + b * a.ks[0] + g * a.ks[2], [&](int r) { return r * a.ks[1]; }, k0, n, a.D, vec);
        load_tile<T, A, TILE, DP>(Vs, static_cast<const T*>(a.v) + b * a.vs[0] + g * a.vs[2], [&](int r) { return r * a.vs[1]; }, k0, n, a.D, vec);
        const T* q = static_cast<const T*>(a.q) + rows.first(a.qs);
        const T* go = static_cast<const T*>(a.dout) + rows.first(a.dos);
        for (int q0 = rank * TILE; q0 < rows.n; q0 += world * TILE) {
            __syncthreads();
            load_tile<T, A, TILE, DP>(Qs, q, [&](int r) { return rows.at(a.qs, r); }, q0, rows.n, a.D, vec);
            load_tile<T, A, TILE, DP>(Gs, go, [&](int r) { return rows.at(a.dos, r); }, q0, rows.n, a.D, vec);
            cp_async_wait<0>();
            __syncthreads();
            A s[M][M] = {}, dp[M][M] = {};
            mul_rows<A, TILE, DP>(s, Qs, Ks, a.D, rows.n - q0, n - k0, ty, tx);
            mul_rows<A, TILE, DP>(dp, Gs, Vs, a.D, rows.n - q0, n - k0, ty, tx);
#pragma unroll
            for (int i = 0; i < M; ++i) {
                const int r = q0 + ty * M + i;
                const A lse = r < rows.n ? static_cast<const A*>(a.lse)[rows.stat(r)] * A(LOG2E) : A(0);
                const A dl = r < rows.n ? static_cast<const A*>(a.delta)[rows.stat(r)] : A(0);
#pragma unroll
                for (int j = 0; j < M; ++j) {
                    const A p = r < rows.n && k0 + tx + 16 * j < n ? exp_acc(s[i][j] * c - lse) : A(0);
                    Ps[(ty * M + i) * LP + tx + 16 * j] = p;
                    Ss[(ty * M + i) * LP + tx + 16 * j] = p * (dp[i][j] - dl);
                }
            }
            __syncthreads();
            mul_cols_t<A, TILE, DP>(dv, Ps, Gs, rows.n - q0, n - k0, ty, tx);
            mul_cols_t<A, TILE, DP>(dk, Ss, Qs, rows.n - q0, n - k0, ty, tx);
        }
    }
    cp_async_wait<0>();
    const int64_t base = (int64_t(b) * a.Lk * a.Hkv + g) * a.D;
    auto at = [&](int r) { return int64_t(r) * a.Hkv * a.D; };
    if (world == 1) {
        store_rows<T, A, TILE, DP>(static_cast<T*>(a.dk) + base, at, k0, a.Lk, a.D, dk, fk, ty, tx);
        store_rows<T, A, TILE, DP>(static_cast<T*>(a.dv) + base, at, k0, a.Lk, a.D, dv, fv, ty, tx);
        return;
    }
    __syncthreads();
    leave_rows<A, TILE, DP>(Qs, dk, ty, tx);
    leave_rows<A, TILE, DP>(Gs, dv, ty, tx);
    cluster.sync();
    store_shared<T, A, TILE, DP>(cluster, static_cast<T*>(a.dk) + base, at, k0, a.Lk, a.D, Qs, A(a.scale));
    store_shared<T, A, TILE, DP>(cluster, static_cast<T*>(a.dv) + base, at, k0, a.Lk, a.D, Gs, A(1));
    cluster.sync();                        // nobody leaves while its shared memory is read
}

// ---------------------------------------------------------------------------

template <typename A>
constexpr int tile_bytes(int tile, int dp) { return tile * (dp + VecOf<A>::N) * int(sizeof(A)); }
template <typename A>
constexpr int score_bytes(int tile) { return tile * (tile + VecOf<A>::N) * int(sizeof(A)); }

constexpr int SMEM_MAX = 227 * 1024;
// the largest tile of scores whose operands fit the shared memory of an SM
template <typename A>
constexpr int fwd_tile(int dp) {
    for (int t : {64, 32})
        if (3 * tile_bytes<A>(t, dp) + score_bytes<A>(t) <= SMEM_MAX) return t;
    return 16;
}
// Float and double problems that come here have few tiles: 32 rows, two blocks an SM with up to 128 float or 64 double
// channels (18 x 1618 x 8 x 2 x 2 x 128 float: 681 us with 64 rows, 392 with 32).
template <typename T>
constexpr int bwd_tile(int dp) {
    using A = typename AccOf<T>::type;
    for (int t : {64, 32})
        if (!(t == 64 && sizeof(T) >= 4) && 4 * tile_bytes<A>(t, dp) + 2 * score_bytes<A>(t) <= SMEM_MAX) return t;
    return 16;
}

// `per_sm`: blocks an SM holds.  `steps`: tiles a block walks over; where there are few blocks a cluster of up to 16 shares them, two each at least
template <typename K>
int launch(K kernel, int64_t units, int64_t steps, int smem, int per_sm, cudaStream_t st, const AttnArgs& a, bool vec) {
    if (units <= 0) return NNVB_OK;
    const int sms = sm_count();
    int world = 1;
    while (world < 16 && units * world * 2 <= int64_t(sms) * per_sm && world * 4 <= steps) world *= 2;
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

bool rows16(const void* p, const int64_t (&s)[3], int64_t esize) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] * esize % 16 == 0 && s[1] * esize % 16 == 0 &&
           s[2] * esize % 16 == 0;
}

template <typename T, int DP>
int forward_t(cudaStream_t st, const AttnArgs& a) {
    using A = typename AccOf<T>::type;
    constexpr int TILE = fwd_tile<A>(DP);
    const bool vec = a.D * sizeof(T) % 16 == 0 && rows16(a.q, a.qs, sizeof(T)) && rows16(a.k, a.ks, sizeof(T)) &&
                     rows16(a.v, a.vs, sizeof(T));
    return launch(attn_fwd_simt_kernel<T, TILE, DP>, ceil_div(int64_t(a.Lq) * (a.Hq / a.Hkv), TILE) * a.Hkv * a.B, 0,
                  3 * tile_bytes<A>(TILE, DP) + score_bytes<A>(TILE), 1, st, a, vec);
}

template <typename T, int DP, int TILE>
int backward_tiles(cudaStream_t st, const AttnArgs& a) {
    using A = typename AccOf<T>::type;
    const bool vec = a.D * sizeof(T) % 16 == 0 && rows16(a.q, a.qs, sizeof(T)) && rows16(a.k, a.ks, sizeof(T)) &&
                     rows16(a.v, a.vs, sizeof(T)) && rows16(a.dout, a.dos, sizeof(T));
    constexpr int SMEM = 4 * tile_bytes<A>(TILE, DP) + 2 * score_bytes<A>(TILE), PER_SM = SMEM <= SMEM_MAX / 2 ? 2 : 1;
    const int64_t tq = ceil_div(int64_t(a.Lq) * (a.Hq / a.Hkv), TILE), tk = ceil_div(a.Lk, TILE), heads = int64_t(a.Hkv) * a.B;
    NNVB_TRY(launch(attn_dq_simt_kernel<T, TILE, DP>, tq * heads, tk, SMEM, PER_SM, st, a, vec));
    return launch(attn_dkv_simt_kernel<T, TILE, DP>, tk * heads, tq, SMEM, PER_SM, st, a, vec);
}

// 128 double channels leave room for two blocks with 16 rows, which suits a side no longer (13 x 239 x 13 x 16 x 2 x 96: 716 us
// with 32 rows, 524 with 16; 14 x 1686 x 21 x 2 x 128: 373 and 527)
template <typename T, int DP>
int backward_t(cudaStream_t st, const AttnArgs& a) {
    if constexpr (sizeof(T) == 8 && DP == 128)
        if (std::min<int64_t>(a.Lk, int64_t(a.Lq) * (a.Hq / a.Hkv)) <= 16) return backward_tiles<T, DP, 16>(st, a);
    return backward_tiles<T, DP, bwd_tile<T>(DP)>(st, a);
}

template <typename T>
int by_head(cudaStream_t st, const AttnArgs& a, bool backward) {
    if (a.D <= 128 && backward) return a.D <= 64 ? backward_t<T, 64>(st, a) : backward_t<T, 128>(st, a);
    if constexpr (sizeof(T) == 2)          // float and double forward: attention_wide.cu
        if (a.D <= 128) return a.D <= 64 ? forward_t<T, 64>(st, a) : forward_t<T, 128>(st, a);
    return backward ? backward_t<T, 256>(st, a) : forward_t<T, 256>(st, a);
}

int by_type(cudaStream_t st, const AttnArgs& a, bool backward) {
    switch (a.dtype) {
        case NNVB_F64: return by_head<double>(st, a, backward);
        case NNVB_F32: return by_head<float>(st, a, backward);
        case NNVB_BF16: return by_head<__nv_bfloat16>(st, a, backward);
        default: return by_head<__half>(st, a, backward);
    }
}

}  // namespace

int attn_forward_simt(cudaStream_t st, const AttnArgs& a) { return by_type(st, a, false); }
int attn_backward_simt(cudaStream_t st, const AttnArgs& a) { return by_type(st, a, true); }

int attn_delta(cudaStream_t st, const AttnArgs& a) {
    const int64_t rows = int64_t(a.B) * a.Lq * a.Hq;
    if (rows == 0) return NNVB_OK;
    const int64_t blocks = ceil_div(rows, 8);
    NNVB_REQUIRE(blocks < (int64_t(1) << 31), "nnvb_cross_attention_backward: too many rows (%lld)", (long long)rows);
    switch (a.dtype) {
        case NNVB_F64: attn_delta_kernel<double><<<unsigned(blocks), 256, 0, st>>>(a); break;
        case NNVB_F32: attn_delta_kernel<float><<<unsigned(blocks), 256, 0, st>>>(a); break;
        case NNVB_BF16: attn_delta_kernel<__nv_bfloat16><<<unsigned(blocks), 256, 0, st>>>(a); break;
        default: attn_delta_kernel<__half><<<unsigned(blocks), 256, 0, st>>>(a); break;
    }
    NNVB_CUDA(cudaGetLastError());
    return NNVB_OK;
}

}  // namespace nnvb
