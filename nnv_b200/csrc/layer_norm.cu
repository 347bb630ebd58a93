// Layer normalisation over the columns of a matrix of rows, and its gradients.
//
//   forward   mu = mean_j x_j,  r = 1 / sqrt(mean_j (x_j - mu)^2 + eps),  z = (x - mu) r,  y = z * scale + offset
//   backward  g = dy * scale,   dx = r (g - mean_j g - z mean_j(g z)),
//             dscale = sum_rows dy z,   doffset = sum_rows dy
//
// Both directions have memory as their floor: forward reads x and writes y, backward reads x and dy and writes dx.  So the rows
// pass through shared memory: blocks stay on the SMs and walk over tiles of rows, and the copy engine (cp.async.bulk)
// keeps the tiles ahead on their way while a tile is worked on, whatever the arithmetic waits for.  A tile of dense rows
// is one copy, so rows of any width move at full speed; rows that are not whole 16-byte pieces are only read element by
// element from shared memory.
//
// A group of TPR threads (part of a warp up to the block) takes a row, N accesses of VEC elements per thread, and works
// on it in registers: forward the mean and then the squared deviations from it (E[x^2] - mean^2 would lose the
// variance of rows with a large mean), backward the sums of g and g (x - mu).  Groups share nothing but the tiles, so
// a group's barriers stop no other group.  About 16 elements per thread spread what a row costs besides its elements;
// with fewer the instruction issue is the bound, not memory.  A thread keeps its columns for all rows, so the weights,
// and the sums over rows for their gradients, stay in registers; they leave a block as one partial row, and a second
// kernel adds the partial rows in a fixed order: no atomics, the same bits every time.  Small tensors are given to one
// cluster of up to 16 blocks, which adds its blocks' sums in distributed shared memory: one launch and no workspace.
// Sums are held in float (double for double).
//
// Double reaches that floor; in 16 bits a wide row's sums in series are the bound, with one row in work an SM (HBM at 0.44 of
// its nominal peak, 1.9 instructions a cycle).  16384 x 8192 bf16: forward 133 us (4.0 TB/s), backward 189 us (4.3 TB/s); 197000 x 192 double: forward 106 us (5.7 TB/s; a copy
// has 6.55).  8 x 768 bf16: 10 us a call, the issue from the host.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "mma_f64.cuh"
#include "tensor_types.cuh"

namespace cg = cooperative_groups;

namespace nnvb {
namespace {

template <typename A>
__device__ __forceinline__ A warp_sum(A x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o, 32);
    return x;
}

// Sums of K values over the TPR threads of a group, the same bits in each of them.  `red` holds a value per warp and
// sum, in two halves that take turns, so that one barrier among the group's warps per call suffices.
template <int TPR, int K, typename A>
__device__ __forceinline__ void group_sum(A (&v)[K], A (*red)[32], int& flip) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o, 32);
    if constexpr (TPR > 32) {
        constexpr int W = TPR / 32, V = W * sizeof(A) < 16 ? W : 16 / sizeof(A);
        const int warp = threadIdx.x / 32, w0 = warp / W * W;
        A(*r)[32] = red + flip;
        flip ^= 2;
        if (threadIdx.x % 32 == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) r[k][warp] = v[k];
        named_bar_sync(1 + warp / W, TPR);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            v[k] = 0;
#pragma unroll
            for (int i = 0; i < W; i += V) {
                const auto q = *reinterpret_cast<const Pack<A, V>*>(&r[k][w0 + i]);
#pragma unroll
                for (int e = 0; e < V; ++e) v[k] += q.v[e];
            }
        }
    }
}
template <int TPR, typename A>
__device__ __forceinline__ A group_sum1(A x, A (*red)[32], int& flip) {
    A v[1] = {x};
    group_sum<TPR>(v, red, flip);
    return v[0];
}

// Makes the compiler forget what it has derived from 16-bit elements: converting them again is one instruction each,
// keeping the converted values as well costs three times the registers.
template <typename T, int VEC>
__device__ __forceinline__ void ln_forget(Pack<T, VEC>& p) {
    if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
        uint32_t* w = reinterpret_cast<uint32_t*>(&p);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) asm volatile("" : "+r"(w[i]));
    }
}

constexpr int LN_THREADS = 512;
constexpr int LN_STAGES = 3;

// How the rows of a tile reach shared memory: as one copy (dense rows), one copy a row (rows of whole 16-byte pieces that
// lie apart), or by plain loads (anything else).
enum { LN_RANGE = 0, LN_BY_ROW = 1, LN_PLAIN = 2 };

struct LnTile {
    int64_t rows, n_tiles;
    int64_t ldx, lddy, ldo;
    const void *x, *dy, *scale, *offset;
    void *out, *mean, *rstd, *partial;
    double eps;
    int cols;
    int R, tensor_bytes;                         // rows of a tile; bytes of one tensor's rows in a stage
    int mode;
    void *dscale, *doffset;                      // one cluster of blocks: where it writes the weights' gradients itself
    int* gave_up;                                // set to 1 when a bounded wait ran out; may be NULL
};

template <typename T, int VEC, int TPR, int N, bool BWD>
__global__ void __launch_bounds__(LN_THREADS, 1)
ln_tile_kernel(const __grid_constant__ LnTile p) {
    using A = typename AccOf<T>::type;
    using P = Pack<T, VEC>;
    constexpr int GROUPS = LN_THREADS / TPR;
    constexpr bool AGAIN = N * VEC * sizeof(A) > 64;       // wide rows: 16-bit values are converted again, not kept
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ uint64_t full[LN_STAGES], empty[LN_STAGES];
    __shared__ int abort_flag, asked[LN_STAGES];           // requests of a stage
    __shared__ __align__(16) A red[4][32];
    const int tid = threadIdx.x;
    const int cols = p.cols, R = p.R;
    const int stage_bytes = p.tensor_bytes * (BWD ? 2 : 1);
    const T *x = static_cast<const T*>(p.x), *dy = static_cast<const T*>(p.dy);
    const int64_t pitch = int64_t(cols) * sizeof(T);

    auto rows_of = [&](int64_t tile) { return int(p.rows - tile * R < R ? p.rows - tile * R : R); };
    // bytes before the first row of a tile in its stage
    auto lead = [&](int64_t tile) { return VEC == 1 && p.mode == LN_RANGE ? int(uint32_t(tile * R * pitch) % 16) : 0; };
    // Bytes that one tensor's copy of a tile moves.  A range runs from the boundary before its first row to the one behind
    // its last, but not past the last boundary inside the tensor: what lies behind that is loaded apart.
    auto bytes_of = [&](int64_t tile) {
        if (VEC > 1 || p.mode != LN_RANGE) return uint32_t(rows_of(tile) * pitch);
        const int64_t from = tile * R * pitch / 16 * 16, to = (tile * R + rows_of(tile)) * pitch, last = p.rows * pitch / 16 * 16;
        const int64_t end = (to + 15) / 16 * 16 < last ? (to + 15) / 16 * 16 : last;
        return uint32_t(end > from ? end - from : 0);
    };
    auto copy = [&](const T* src, int64_t ld, int64_t tile, unsigned char* dst, uint64_t* bar) {
        if (p.mode == LN_RANGE) {
            const uint32_t bytes = bytes_of(tile);
            if (bytes) bulk_copy_g2s(dst, reinterpret_cast<const char*>(src) + tile * R * pitch / 16 * 16, bytes, bar);
        } else {
            for (int r = 0; r < rows_of(tile); ++r) bulk_copy_g2s(dst + r * pitch, src + (tile * R + r) * ld, uint32_t(pitch), bar);
        }
    };
    auto request = [&](int64_t tile, int s) {              // one thread
        ++asked[s];
        unsigned char* dst = ring + s * stage_bytes;
        mbar_expect_bytes(&full[s], bytes_of(tile) * (BWD ? 2 : 1));
        copy(x, p.ldx, tile, dst, &full[s]);
        if (BWD) copy(dy, p.lddy, tile, dst + p.tensor_bytes, &full[s]);
    };

    if (tid == 0) {
        abort_flag = 0;
        for (int s = 0; s < LN_STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], LN_THREADS / 32); asked[s] = 0; }
        mbar_init_fence();
        if (p.mode != LN_PLAIN)
            for (int s = 0; s < LN_STAGES; ++s)
                if (blockIdx.x + int64_t(s) * gridDim.x < p.n_tiles) request(blockIdx.x + int64_t(s) * gridDim.x, s);
    }

    const int t = tid % TPR, grp = tid / TPR;
    P sc[N], of[N];
    // elements are worked on in pairs (one instruction for two floats) where an access holds pairs
    constexpr int UN = VEC > 1 ? 2 : 1, H = VEC / UN;
    using U = typename std::conditional<VEC == 1, A, Pair<A>>::type;
    auto one = [](A x) { if constexpr (VEC == 1) return x; else return Pair<A>{x, x}; };
    auto unit = [](const P& v, int e) {
        if constexpr (VEC == 1) return A(to_acc(v.v[0]));
        else return Pair<A>{A(to_acc(v.v[e])), A(to_acc(v.v[e + 1]))};
    };
    auto put = [](P& o, int e, U z) {
        if constexpr (VEC == 1) o.v[0] = from_acc<T, A>(z);
        else {
            o.v[e] = from_acc<T, A>(z.x);
            o.v[e + 1] = from_acc<T, A>(z.y);
        }
    };
    U acc_s[BWD ? N * H : 1], acc_o[BWD ? N * H : 1];
    const bool has_s = p.scale != nullptr, has_o = !BWD && p.offset != nullptr;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int c = (t + i * TPR) * VEC;
        if (c < cols) {
            if (has_s) sc[i] = *reinterpret_cast<const P*>(static_cast<const T*>(p.scale) + c);
            if constexpr (!BWD)
                if (has_o) of[i] = *reinterpret_cast<const P*>(static_cast<const T*>(p.offset) + c);
        }
    }
#pragma unroll
    for (int f = 0; f < (BWD ? N * H : 1); ++f) acc_s[f] = acc_o[f] = one(0);
    __syncthreads();

    const A inv_n = A(1) / A(cols), eps = A(p.eps);
    int flip = 0, s = 0;
    uint32_t phase = 0;
    bool ok = true;
    // A failed wait changes no control flow: the groups' barriers need every thread.  Its thread adds NaN to its group's
    // sums, so the row's results and statistics become NaN whatever the others of the group have seen.
    for (int64_t tile = blockIdx.x; tile < p.n_tiles; tile += gridDim.x) {
        unsigned char* st = ring + s * stage_bytes;
        const int n = rows_of(tile);
        const int64_t row0 = tile * R;
        if (p.mode == LN_PLAIN) {
            __syncthreads();
            for (int i = tid; i < n * cols; i += LN_THREADS) {
                const int r = i / cols, c = i % cols;
                reinterpret_cast<T*>(st)[i] = x[(row0 + r) * p.ldx + c];
                if (BWD) reinterpret_cast<T*>(st + p.tensor_bytes)[i] = dy[(row0 + r) * p.lddy + c];
            }
            __syncthreads();
        } else {
            ok = ok && mbar_wait_or_abort(&full[s], phase, &abort_flag);
            if (VEC == 1 && p.mode == LN_RANGE && tile + 8 >= p.n_tiles) {       // under 16 bytes: at most 7 tiles of one element
                const int64_t all = n * pitch, got = int64_t(bytes_of(tile)) - lead(tile);
                const int left = int((all - (got > 0 ? (got < all ? got : all) : 0)) / int(sizeof(T)));
                if (left > 0) {                 // the tensor's last elements
                    if (tid < left) {
                        const int64_t at = int64_t(n) * cols - left + tid;
                        reinterpret_cast<T*>(st + lead(tile))[at] = x[row0 * cols + at];
                        if (BWD) reinterpret_cast<T*>(st + p.tensor_bytes + lead(tile))[at] = dy[row0 * cols + at];
                    }
                    __syncthreads();
                }
            }
        }
        const T* sx = reinterpret_cast<const T*>(st + lead(tile)) + grp * cols;
        const T* sg = reinterpret_cast<const T*>(st + p.tensor_bytes + lead(tile)) + grp * cols;
        T* out = static_cast<T*>(p.out) + (row0 + grp) * p.ldo;
        for (int base = 0; base < n; base += GROUPS, sx += GROUPS * cols, sg += GROUPS * cols, out += GROUPS * p.ldo) {
            const int64_t row = row0 + base + grp;
            const bool live = base + grp < n;
            if (TPR >= 32 && !live) break;      // groups of whole warps go on to the next tile
            P px[N];
            auto has = [&](int i) { return live && (t + i * TPR) * VEC < cols; };
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (has(i)) px[i] = *reinterpret_cast<const P*>(sx + (t + i * TPR) * VEC);
            if constexpr (!BWD) {
                U sum = one(ok ? A(0) : A(NAN));
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (has(i))
#pragma unroll
                        for (int e = 0; e < VEC; e += UN) sum = add2(sum, unit(px[i], e));
                const A mean = group_sum1<TPR>(across(sum), red, flip) * inv_n;
                U dev = one(0);
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (has(i)) {
                        if (AGAIN) ln_forget(px[i]);
#pragma unroll
                        for (int e = 0; e < VEC; e += UN) {
                            const U d = add2(unit(px[i], e), one(-mean));
                            dev = fma2(d, d, dev);
                        }
                    }
                const A rstd = rsqrt_acc(group_sum1<TPR>(across(dev), red, flip) * inv_n + eps);
                if (live && t == 0) {
                    if (p.mean) static_cast<A*>(p.mean)[row] = mean;
                    if (p.rstd) static_cast<A*>(p.rstd)[row] = rstd;
                }
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (has(i)) {
                        P o;
                        if (AGAIN) {
                            ln_forget(px[i]);
                            if (has_s) ln_forget(sc[i]);
                            if (has_o) ln_forget(of[i]);
                        }
#pragma unroll
                        for (int e = 0; e < VEC; e += UN) {
                            U z = mul2(add2(unit(px[i], e), one(-mean)), one(rstd));
                            if (has_s) z = has_o ? fma2(z, unit(sc[i], e), unit(of[i], e)) : mul2(z, unit(sc[i], e));
                            else if (has_o) z = add2(z, unit(of[i], e));
                            put(o, e, z);
                        }
                        *reinterpret_cast<P*>(out + (t + i * TPR) * VEC) = o;
                    }
            } else {
                P pg[N];
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (has(i)) pg[i] = *reinterpret_cast<const P*>(sg + (t + i * TPR) * VEC);
                const A mu = live ? __ldg(static_cast<const A*>(p.mean) + row) : A(0);
                const A rs = live ? __ldg(static_cast<const A*>(p.rstd) + row) : A(0);
                U s1 = one(ok ? A(0) : A(NAN)), s2 = s1;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (has(i)) {
                        if (AGAIN && has_s) ln_forget(sc[i]);
#pragma unroll
                        for (int e = 0; e < VEC; e += UN) {
                            const U d = unit(pg[i], e), g = has_s ? mul2(d, unit(sc[i], e)) : d;
                            s1 = add2(s1, g);
                            s2 = fma2(g, add2(unit(px[i], e), one(-mu)), s2);
                        }
                    }
                A sums[2] = {across(s1), across(s2)};
                group_sum<TPR>(sums, red, flip);
                const A k1 = -sums[0] * inv_n * rs, k2 = -sums[1] * inv_n * rs * rs * rs;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (has(i)) {
                        P o;
                        if (AGAIN) {
                            ln_forget(px[i]);
                            ln_forget(pg[i]);
                            if (has_s) ln_forget(sc[i]);
                        }
#pragma unroll
                        for (int e = 0; e < VEC; e += UN) {
                            const U xc = add2(unit(px[i], e), one(-mu)), d = unit(pg[i], e), dr = mul2(d, one(rs));
                            U &as = acc_s[i * H + e / UN], &ao = acc_o[i * H + e / UN];
                            as = fma2(dr, xc, as);
                            ao = add2(ao, d);
                            const U k = fma2(xc, one(k2), one(k1));
                            put(o, e, has_s ? fma2(dr, unit(sc[i], e), k) : add2(dr, k));
                        }
                        *reinterpret_cast<P*>(out + (t + i * TPR) * VEC) = o;
                    }
            }
        }
        if (p.mode != LN_PLAIN) {
            __syncwarp();
            if (tid % 32 == 0) mbar_arrive(&empty[s]);
            // The stage of the tile before is requested again now: by this time the other warps are through with it, so
            // the thread that asks hardly waits.
            if (tid == 0 && tile != int64_t(blockIdx.x)) {
                const int64_t next = tile + int64_t(LN_STAGES - 1) * gridDim.x;
                const int sp = s ? s - 1 : LN_STAGES - 1;
                if (next < p.n_tiles && ok) {
                    ok = mbar_wait_or_abort(&empty[sp], s ? phase : phase ^ 1, &abort_flag);
                    async_proxy_fence();
                    if (ok) request(next, sp);
                }
            }
        }
        if (++s == LN_STAGES) { s = 0; phase ^= 1; }
    }
    if (!ok && p.gave_up) *p.gave_up = 1;
    if (!ok && tid == 0)                        // gave up: copies may still be on their way into this block's memory
        for (int i = 0; i < LN_STAGES; ++i)
            if (asked[i] > 0) mbar_wait(&full[i], (asked[i] - 1) & 1, 1 << 20);

    if constexpr (BWD) {
        const bool whole = p.dscale || p.doffset;
        if (!p.partial && !whole) return;
        // the groups' sums, added in group order, one access of columns at a time through the ring
        A* buf = reinterpret_cast<A*>(ring);
        A* own = buf + LN_THREADS * VEC;        // a cluster's blocks keep their sums in shared memory, behind that
        A* ps = whole ? own : static_cast<A*>(p.partial) + int64_t(blockIdx.x) * 2 * cols;
        const A bad = ok ? A(0) : A(NAN);
#pragma unroll
        for (int k = 0; k < 2 * N; ++k) {
            const int i = k >> 1;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const U a = (k & 1) ? acc_o[i * H + e / UN] : acc_s[i * H + e / UN];
                if constexpr (VEC == 1) buf[tid] = a + bad;
                else buf[tid * VEC + e] = (e % 2 ? a.y : a.x) + bad;
            }
            __syncthreads();
            for (int j = tid; j < TPR * VEC; j += LN_THREADS) {
                const int c = i * TPR * VEC + j;
                if (c < cols) {
                    A sum = 0;
                    for (int g = 0; g < GROUPS; ++g) sum += buf[g * TPR * VEC + j];
                    ps[(k & 1) * int64_t(cols) + c] = sum;
                }
            }
        }
        if (whole) {
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();
            const int rank = int(cluster.block_rank()), world = int(cluster.num_blocks());
            for (int c = rank * LN_THREADS + tid; c < 2 * cols; c += world * LN_THREADS) {
                A sum = 0;
                for (int w = 0; w < world; ++w) sum += *cluster.map_shared_rank(own + c, w);
                T* to = static_cast<T*>(c < cols ? p.dscale : p.doffset);
                if (to) to[c < cols ? c : c - cols] = from_acc<T, A>(sum);
            }
            cluster.sync();                     // nobody leaves while its shared memory is read
        }
    }
}

// Rows wider than the registers of a block: the same sums with the row read again (from L2) for each of them.
template <typename T>
__global__ void __launch_bounds__(1024)
ln_forward_wide_kernel(int64_t cols, const T* __restrict__ x, int64_t ldx, const T* __restrict__ scale,
                       const T* __restrict__ offset, typename AccOf<T>::type eps, T* __restrict__ y, int64_t ldy,
                       typename AccOf<T>::type* __restrict__ mean_out, typename AccOf<T>::type* __restrict__ rstd_out) {
    using A = typename AccOf<T>::type;
    __shared__ __align__(16) A red[4][32];
    int flip = 0;
    const int64_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    A s = 0;
    for (int64_t c = threadIdx.x; c < cols; c += 1024) s += to_acc(xr[c]);
    const A inv_n = A(1) / A(cols);
    const A mean = group_sum1<1024>(s, red, flip) * inv_n;
    A q = 0;
    for (int64_t c = threadIdx.x; c < cols; c += 1024) {
        const A d = to_acc(xr[c]) - mean;
        q += d * d;
    }
    const A rstd = rsqrt_acc(group_sum1<1024>(q, red, flip) * inv_n + eps);
    if (threadIdx.x == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
    T* yr = y + row * ldy;
    for (int64_t c = threadIdx.x; c < cols; c += 1024) {
        A z = (to_acc(xr[c]) - mean) * rstd;
        if (scale) z *= to_acc(scale[c]);
        if (offset) z += to_acc(offset[c]);
        yr[c] = from_acc<T, A>(z);
    }
}

// dscale / doffset: partial rows added in order, 32 columns per block, the rows over 32 warps
template <typename T>
__global__ void __launch_bounds__(1024)
ln_reduce_kernel(int n_parts, int64_t cols, const typename AccOf<T>::type* __restrict__ partial, T* __restrict__ dscale,
                 T* __restrict__ doffset) {
    using A = typename AccOf<T>::type;
    __shared__ A buf[32][33];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t c = int64_t(blockIdx.x) * 32 + lane;      // 0 .. 2 * cols
    A s = 0;
    if (c < 2 * cols)
#pragma unroll 8
        for (int p = warp; p < n_parts; p += 32) s += partial[int64_t(p) * 2 * cols + c];
    buf[warp][lane] = s;
    __syncthreads();
    // warp w adds column w over the 32 warps, in the order of the shuffles
    s = warp_sum(buf[lane][warp]);
    const int64_t cw = int64_t(blockIdx.x) * 32 + warp;
    if (lane == 0 && cw < 2 * cols) {
        T* out = cw < cols ? dscale : doffset;
        if (out) out[cw < cols ? cw : cw - cols] = from_acc<T, A>(s);
    }
}

// Wide rows, backward: dx by one block per row; the weights' partial sums by a kernel over columns and row slices.
template <typename T>
__global__ void __launch_bounds__(1024)
ln_backward_wide_kernel(int64_t cols, const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                        const T* __restrict__ scale, const typename AccOf<T>::type* __restrict__ mean,
                        const typename AccOf<T>::type* __restrict__ rstd, T* __restrict__ dx, int64_t lddx) {
    using A = typename AccOf<T>::type;
    __shared__ __align__(16) A red[4][32];
    int flip = 0;
    const int64_t row = blockIdx.x;
    const T *xr = x + row * ldx, *gr = dy + row * lddy;
    const A mu = mean[row], r = rstd[row];
    A s1 = 0, s2 = 0;
    for (int64_t c = threadIdx.x; c < cols; c += 1024) {
        const A z = (to_acc(xr[c]) - mu) * r;
        const A g = scale ? to_acc(gr[c]) * to_acc(scale[c]) : to_acc(gr[c]);
        s1 += g;
        s2 += g * z;
    }
    A sums[2] = {s1, s2};
    group_sum<1024>(sums, red, flip);
    const A m1 = sums[0] / A(cols), m2 = sums[1] / A(cols);
    for (int64_t c = threadIdx.x; c < cols; c += 1024) {
        const A z = (to_acc(xr[c]) - mu) * r;
        const A g = scale ? to_acc(gr[c]) * to_acc(scale[c]) : to_acc(gr[c]);
        dx[row * lddx + c] = from_acc<T, A>(r * (g - m1 - z * m2));
    }
}

template <typename T>
__global__ void __launch_bounds__(256)
ln_weights_wide_kernel(int64_t rows, int64_t cols, const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x,
                       int64_t ldx, const typename AccOf<T>::type* __restrict__ mean,
                       const typename AccOf<T>::type* __restrict__ rstd, typename AccOf<T>::type* __restrict__ partial) {
    using A = typename AccOf<T>::type;
    const int64_t c = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (c >= cols) return;
    A s = 0, o = 0;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const A d = to_acc(dy[row * lddy + c]);
        s += d * ((to_acc(x[row * ldx + c]) - mean[row]) * rstd[row]);
        o += d;
    }
    partial[int64_t(blockIdx.y) * 2 * cols + c] = s;
    partial[int64_t(blockIdx.y) * 2 * cols + cols + c] = o;
}

// ---------------------------------------------------------------------------
// host side

struct LnArgs {
    cudaStream_t st;
    int64_t rows, cols;
    const void *dy, *x, *scale, *offset;
    int64_t lddy, ldx, ldo;
    double eps;
    void *out, *mean, *rstd;
    void* partial;
    int grid;               // backward: blocks
    void *dscale, *doffset;
    int* gave_up;
};

// Shared memory that any call may need: every stage's tiles, or a cluster's sums.  The limit of a kernel belongs to the
// process, so every call sets this value; with its own need, a call with few rows could lower the limit between another
// thread's setting and its launch.
constexpr int LN_SMEM = 200 * 1024;

constexpr int LN_MAX_PARTS = 2 * 148;        // partial rows of the weights' gradients: the most slices of rows (wide rows)

// Backward of tensors up to this size runs in one cluster: its 16 SMs take about as long as a second launch does.
bool ln_in_cluster(int64_t rows, int64_t cols) { return rows * cols <= 512 * 1024 && cols <= 4096; }

template <typename T, int VEC, int TPR, int N, bool BWD>
int ln_tile(LnArgs& a, int mode) {
    constexpr int GROUPS = LN_THREADS / TPR, TENSORS = BWD ? 2 : 1;
    const bool cluster = BWD && (a.dscale || a.doffset) && ln_in_cluster(a.rows, a.cols);
    const int64_t slots = cluster ? 16 : std::min(sm_count(), 148);
    const int64_t pitch = a.cols * int64_t(sizeof(T));
    LnTile p{};
    p.rows = a.rows; p.cols = int(a.cols);
    p.ldx = a.ldx; p.lddy = a.lddy; p.ldo = a.ldo;
    p.x = a.x; p.dy = a.dy; p.scale = a.scale; p.offset = a.offset;
    p.out = a.out; p.mean = a.mean; p.rstd = a.rstd; p.partial = a.partial;
    p.eps = a.eps;
    p.mode = mode;
    p.gave_up = a.gave_up;
    // as many rounds of all groups as a stage holds, but no more rows than spread over all blocks
    const int64_t budget = LN_SMEM / LN_STAGES;
    int64_t R = (budget - 32 * TENSORS - 256) / (TENSORS * pitch);
    R = std::min<int64_t>(R, ceil_div(a.rows, slots));
    R = R >= GROUPS ? R / GROUPS * GROUPS : std::max<int64_t>(R, 1);
    p.R = int(R);
    p.n_tiles = ceil_div(a.rows, R);
    p.tensor_bytes = int(round_up(R * pitch + 32, 128));
    using A = typename AccOf<T>::type;
    const int sums = BWD ? (LN_THREADS * VEC + (cluster ? 2 * p.cols : 0)) * int(sizeof(A)) : 0;
    const int smem = std::max<int>(LN_STAGES * p.tensor_bytes * TENSORS, sums);
    a.grid = int(std::min<int64_t>(p.n_tiles, slots));
    auto kernel = ln_tile_kernel<T, VEC, TPR, N, BWD>;
    NNVB_REQUIRE(smem <= LN_SMEM, "nnvb_layer_norm: rows of %lld columns need %d bytes of shared memory", (long long)a.cols, smem);
    NNVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LN_SMEM));
    if (cluster) {
        int world = 1;
        while (world < a.grid) world *= 2;
        p.dscale = a.dscale; p.doffset = a.doffset;
        if (world > 8) NNVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(unsigned(world));
        cfg.blockDim = dim3(LN_THREADS);
        cfg.dynamicSmemBytes = size_t(smem);
        cfg.stream = a.st;
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = unsigned(world);
        at.val.clusterDim.y = at.val.clusterDim.z = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        NNVB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
        return NNVB_OK;
    }
    kernel<<<unsigned(a.grid), LN_THREADS, smem, a.st>>>(p);
    NNVB_CUDA(cudaGetLastError());
    return NNVB_OK;
}

// The narrowest group that holds the columns with about 16 elements (8 doubles) per thread.
template <typename T, int VEC, bool BWD>
int ln_by_width(LnArgs& a, int mode, bool* done) {
    constexpr int E = sizeof(T) == 8 ? 8 : 16, N = E / VEC;
    const int64_t c = a.cols;
    *done = true;
    if (c <= 8 * E / 2) return ln_tile<T, VEC, 8, N / 2, BWD>(a, mode);
    if (c <= 8 * E) return ln_tile<T, VEC, 8, N, BWD>(a, mode);
    if (c <= 32 * E / 2) return ln_tile<T, VEC, 32, N / 2, BWD>(a, mode);
    if (c <= 32 * E) return ln_tile<T, VEC, 32, N, BWD>(a, mode);
    if (c <= 64 * E) return ln_tile<T, VEC, 64, N, BWD>(a, mode);
    if (c <= 128 * E) return ln_tile<T, VEC, 128, N, BWD>(a, mode);
    if (c <= 256 * E) return ln_tile<T, VEC, 256, N, BWD>(a, mode);
    if (c <= 512 * E) return ln_tile<T, VEC, 512, N, BWD>(a, mode);
    // the ring holds a row per stage at least
    const int64_t row = round_up(c * int64_t(sizeof(T)) + 32, 128) * (BWD ? 2 : 1);
    if (c <= 512 * 2 * E && row * LN_STAGES <= LN_SMEM) return ln_tile<T, VEC, 512, 2 * N, BWD>(a, mode);
    *done = false;
    return NNVB_OK;
}

// Whether all rows are whole 16-byte pieces on 16-byte boundaries, and how tiles of them are copied.
template <typename T>
void ln_access(const LnArgs& a, bool bwd, bool* vec, int* mode) {
    constexpr int64_t V = 16 / sizeof(T);
    auto on16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool base = on16(a.x) && (!bwd || on16(a.dy));
    const bool pieces = base && a.cols % V == 0 && a.ldx % V == 0 && (!bwd || a.lddy % V == 0);
    *vec = pieces && on16(a.scale) && on16(a.offset) && on16(a.out) && a.ldo % V == 0;
    if (base && a.ldx == a.cols && (!bwd || a.lddy == a.cols)) *mode = LN_RANGE;
    else *mode = pieces ? LN_BY_ROW : LN_PLAIN;
}

template <typename T, bool BWD>
int ln_run(LnArgs& a, bool* done) {
    bool vec;
    int mode;
    ln_access<T>(a, BWD, &vec, &mode);
    return vec ? ln_by_width<T, 16 / sizeof(T), BWD>(a, mode, done) : ln_by_width<T, 1, BWD>(a, mode, done);
}

template <typename T>
int ln_forward_t(LnArgs a) {
    using A = typename AccOf<T>::type;
    bool done;
    NNVB_TRY((ln_run<T, false>(a, &done)));
    if (done) return NNVB_OK;
    ln_forward_wide_kernel<T><<<unsigned(a.rows), 1024, 0, a.st>>>(
        a.cols, static_cast<const T*>(a.x), a.ldx, static_cast<const T*>(a.scale), static_cast<const T*>(a.offset),
        A(a.eps), static_cast<T*>(a.out), a.ldo, static_cast<A*>(a.mean), static_cast<A*>(a.rstd));
    NNVB_CUDA(cudaGetLastError());
    return NNVB_OK;
}

template <typename T>
int ln_backward_t(LnArgs a, void* dscale, void* doffset) {
    using A = typename AccOf<T>::type;
    bool done;
    a.dscale = dscale; a.doffset = doffset;
    NNVB_TRY((ln_run<T, true>(a, &done)));
    if (!done) {
        ln_backward_wide_kernel<T><<<unsigned(a.rows), 1024, 0, a.st>>>(
            a.cols, static_cast<const T*>(a.dy), a.lddy, static_cast<const T*>(a.x), a.ldx, static_cast<const T*>(a.scale),
            static_cast<const A*>(a.mean), static_cast<const A*>(a.rstd), static_cast<T*>(a.out), a.ldo);
        NNVB_CUDA(cudaGetLastError());
        if (a.partial) {
            const int64_t cb = ceil_div(a.cols, 256);
            a.grid = int(std::max<int64_t>(1, std::min<int64_t>({a.rows, LN_MAX_PARTS, ceil_div(int64_t(sm_count()) * 8, cb)})));
            ln_weights_wide_kernel<T><<<dim3(unsigned(cb), unsigned(a.grid)), 256, 0, a.st>>>(
                a.rows, a.cols, static_cast<const T*>(a.dy), a.lddy, static_cast<const T*>(a.x), a.ldx,
                static_cast<const A*>(a.mean), static_cast<const A*>(a.rstd), static_cast<A*>(a.partial));
            NNVB_CUDA(cudaGetLastError());
        }
    }
    if (a.partial) {
        ln_reduce_kernel<T><<<unsigned(ceil_div(2 * a.cols, 32)), 1024, 0, a.st>>>(
            a.grid, a.cols, static_cast<const A*>(a.partial), static_cast<T*>(dscale), static_cast<T*>(doffset));
        NNVB_CUDA(cudaGetLastError());
    }
    return NNVB_OK;
}

}  // namespace

int sm_count() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

int64_t dtype_bytes(int dtype) {
    switch (dtype) {
        case NNVB_F64: return 8;
        case NNVB_F32: return 4;
        case NNVB_BF16: case NNVB_F16: return 2;
        default: return 0;
    }
}

}  // namespace nnvb

using namespace nnvb;

namespace {

int ln_forward(cudaStream_t st, int dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* scale,
               const void* offset, double eps, void* y, int64_t ldy, void* mean, void* rstd, int* gave_up) {
    NNVB_REQUIRE(dtype_bytes(dtype) > 0, "nnvb_layer_norm_forward: unknown element type %d", dtype);
    NNVB_REQUIRE(rows >= 0 && cols >= 1 && rows < (int64_t(1) << 31) && cols < (int64_t(1) << 31),
                 "nnvb_layer_norm_forward: bad sizes (rows=%lld, cols=%lld)", (long long)rows, (long long)cols);
    NNVB_REQUIRE(ldx >= cols && ldy >= cols, "nnvb_layer_norm_forward: rows overlap (cols=%lld, ldx=%lld, ldy=%lld)",
                 (long long)cols, (long long)ldx, (long long)ldy);
    NNVB_REQUIRE(eps >= 0 && eps < 1e30, "nnvb_layer_norm_forward: eps must be finite and not negative");
    if (rows == 0) return NNVB_OK;
    NNVB_REQUIRE(x && y, "nnvb_layer_norm_forward: NULL pointer");
    LnArgs a{st, rows, cols, nullptr, x, scale, offset, 0, ldx, ldy, eps, y, mean, rstd, nullptr, 0, nullptr, nullptr, gave_up};
    switch (dtype) {
        case NNVB_F64: return ln_forward_t<double>(a);
        case NNVB_F32: return ln_forward_t<float>(a);
        case NNVB_BF16: return ln_forward_t<__nv_bfloat16>(a);
        default: return ln_forward_t<__half>(a);
    }
}

}  // namespace

int nnvb::layer_norm_rows(cudaStream_t st, int64_t rows, int64_t cols, const double* x, int64_t ld, const double* scale,
                          const double* offset, double eps, double* y, int* gave_up) {
    return ln_forward(st, NNVB_F64, rows, cols, x, ld, scale, offset, eps, y, ld, nullptr, nullptr, gave_up);
}

extern "C" {

int nnvb_layer_norm_forward(void* stream, int dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx,
                            const void* scale, const void* offset, double eps, void* y, int64_t ldy, void* mean,
                            void* rstd) {
    return ln_forward(static_cast<cudaStream_t>(stream), dtype, rows, cols, x, ldx, scale, offset, eps, y, ldy, mean, rstd, nullptr);
}

int64_t nnvb_layer_norm_workspace(int dtype, int64_t rows, int64_t cols) {
    if (dtype_bytes(dtype) == 0 || rows < 0 || cols < 1 || ln_in_cluster(rows, cols)) return 0;
    return std::min<int64_t>(std::max<int64_t>(rows, 1), LN_MAX_PARTS) * 2 * cols * (dtype == NNVB_F64 ? 8 : 4);
}

int nnvb_layer_norm_backward(void* stream, int dtype, int64_t rows, int64_t cols, const void* dy, int64_t lddy,
                             const void* x, int64_t ldx, const void* scale, const void* mean, const void* rstd, void* dx,
                             int64_t lddx, void* dscale, void* doffset, void* workspace, int64_t workspace_bytes) {
    NNVB_REQUIRE(dtype_bytes(dtype) > 0, "nnvb_layer_norm_backward: unknown element type %d", dtype);
    NNVB_REQUIRE(rows >= 0 && cols >= 1 && rows < (int64_t(1) << 31) && cols < (int64_t(1) << 31),
                 "nnvb_layer_norm_backward: bad sizes (rows=%lld, cols=%lld)", (long long)rows, (long long)cols);
    NNVB_REQUIRE(lddy >= cols && ldx >= cols && lddx >= cols, "nnvb_layer_norm_backward: rows overlap");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {                       // the sums over no rows
        if (dscale) NNVB_CUDA(cudaMemsetAsync(dscale, 0, size_t(cols * dtype_bytes(dtype)), st));
        if (doffset) NNVB_CUDA(cudaMemsetAsync(doffset, 0, size_t(cols * dtype_bytes(dtype)), st));
        return NNVB_OK;
    }
    NNVB_REQUIRE(dy && x && mean && rstd && dx, "nnvb_layer_norm_backward: NULL pointer");
    const bool weights = (dscale || doffset) && !ln_in_cluster(rows, cols);
    if (weights) {
        NNVB_REQUIRE(workspace && workspace_bytes >= nnvb_layer_norm_workspace(dtype, rows, cols) &&
                         reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                     "nnvb_layer_norm_backward: the weights' gradients need a 16-byte aligned workspace of %lld bytes",
                     (long long)nnvb_layer_norm_workspace(dtype, rows, cols));
    }
    LnArgs a{st, rows, cols, dy, x, scale, nullptr, lddy, ldx, lddx, 0.0, dx, const_cast<void*>(mean),
             const_cast<void*>(rstd), weights ? workspace : nullptr, 0, nullptr, nullptr, nullptr};
    switch (dtype) {
        case NNVB_F64: return ln_backward_t<double>(a, dscale, doffset);
        case NNVB_F32: return ln_backward_t<float>(a, dscale, doffset);
        case NNVB_BF16: return ln_backward_t<__nv_bfloat16>(a, dscale, doffset);
        default: return ln_backward_t<__half>(a, dscale, doffset);
    }
}

}  // extern "C"
