// Layer normalisation over the columns of a matrix of rows, and its gradients.
//
//   forward   mu = mean_j x_j,  r = 1 / sqrt(mean_j (x_j - mu)^2 + eps),  z = (x - mu) r,  y = z * scale + offset
//   backward  g = dy * scale,   dx = r (g - mean_j g - z mean_j(g z)),
//             dscale = sum_rows dy z,   doffset = sum_rows dy
//
// Both directions are bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.  A row
// is read once into the registers of a group of TPR threads (a part of a warp, a warp, or a whole block for wide
// rows), so the mean, the squared deviations and the result all come from one read; the deviations are summed in a
// second pass over registers, because E[x^2] - mean^2 loses the variance of rows with a large mean.  Sums are held
// in float (double for double).
//
// The weights' gradients are sums over the rows.  The backward kernel keeps one CTA (or a few) on every SM that walks
// over rows; a thread holds the same columns for all its rows and sums them in registers, the block adds its
// groups in shared memory and writes one partial row, and a second kernel adds the partial rows in a fixed order:
// no atomics, the same bits every time.
#include <algorithm>
#include <initializer_list>

#include "common.cuh"
#include "tensor_types.cuh"

namespace nnvb {
namespace {

constexpr int LN_BLOCK = 256;           // threads of a block whose rows fit a warp or less

template <typename A>
__device__ __forceinline__ A warp_sum(A x, int width) {
    for (int o = width / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o, 32);
    return x;
}

// Sum of x over the TPR threads of a row, the same bits in each of them.  `red` holds one value per warp of a group;
// two alternating halves let one barrier per call suffice.
template <int TPR, typename A>
__device__ __forceinline__ A group_sum(A x, A* red, int& flip) {
    if constexpr (TPR <= 32) {
        return warp_sum(x, TPR);
    } else {
        constexpr int W = TPR / 32;
        x = warp_sum(x, 32);
        const int warp = threadIdx.x / 32;
        A* r = red + (flip ? 32 : 0);
        flip ^= 1;
        if (threadIdx.x % 32 == 0) r[warp] = x;
        __syncthreads();
        const int w0 = warp / W * W;
        A s = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) s += r[w0 + i];
        return s;
    }
}

template <typename A>
struct Two { A a, b; };

template <int TPR, typename A>
__device__ __forceinline__ Two<A> group_sum2(A x, A y, Two<A>* red, int& flip) {
    if constexpr (TPR <= 32) {
        return {warp_sum(x, TPR), warp_sum(y, TPR)};
    } else {
        constexpr int W = TPR / 32;
        x = warp_sum(x, 32);
        y = warp_sum(y, 32);
        const int warp = threadIdx.x / 32;
        Two<A>* r = red + (flip ? 32 : 0);
        flip ^= 1;
        if (threadIdx.x % 32 == 0) r[warp] = {x, y};
        __syncthreads();
        const int w0 = warp / W * W;
        Two<A> s{0, 0};
#pragma unroll
        for (int i = 0; i < W; ++i) { s.a += r[w0 + i].a; s.b += r[w0 + i].b; }
        return s;
    }
}

// TPR threads per row, NV accesses of VEC elements per thread; TPR * NV * VEC >= cols.
template <typename T, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(TPR > LN_BLOCK ? TPR : LN_BLOCK)
ln_forward_kernel(int64_t rows, int cols, const T* __restrict__ x, int64_t ldx, const T* __restrict__ scale,
                  const T* __restrict__ offset, typename AccOf<T>::type eps, T* __restrict__ y, int64_t ldy,
                  typename AccOf<T>::type* __restrict__ mean_out, typename AccOf<T>::type* __restrict__ rstd_out) {
    using A = typename AccOf<T>::type;
    using P = Pack<T, VEC>;
    constexpr int BLOCK = TPR > LN_BLOCK ? TPR : LN_BLOCK;
    constexpr int RPB = BLOCK / TPR;
    __shared__ A red[64];
    int flip = 0;
    const int t = threadIdx.x % TPR;
    const int64_t row = int64_t(blockIdx.x) * RPB + threadIdx.x / TPR;
    const bool live = row < rows;
    const T* xr = x + (live ? row : 0) * ldx;
    P buf[NV];
    const int c0 = t * VEC;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * TPR * VEC;
        if (c < cols && live) buf[i] = *reinterpret_cast<const P*>(xr + c);
    }
    A s = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (c0 + i * TPR * VEC < cols && live) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) s += to_acc(buf[i].v[e]);
        }
    const A inv_n = A(1) / A(cols);
    const A mean = group_sum<TPR>(s, red, flip) * inv_n;
    A q = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (c0 + i * TPR * VEC < cols && live) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const A d = to_acc(buf[i].v[e]) - mean;
                q += d * d;
            }
        }
    const A rstd = rsqrt_acc(group_sum<TPR>(q, red, flip) * inv_n + eps);
    if (!live) return;
    if (t == 0) {
        if (mean_out) mean_out[row] = mean;
        if (rstd_out) rstd_out[row] = rstd;
    }
    T* yr = y + row * ldy;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * TPR * VEC;
        if (c < cols) {
            P sc, of, o;
            if (scale) sc = *reinterpret_cast<const P*>(scale + c);
            if (offset) of = *reinterpret_cast<const P*>(offset + c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                A z = (to_acc(buf[i].v[e]) - mean) * rstd;
                if (scale) z *= to_acc(sc.v[e]);
                if (offset) z += to_acc(of.v[e]);
                o.v[e] = from_acc<T, A>(z);
            }
            *reinterpret_cast<P*>(yr + c) = o;
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
    __shared__ A red[64];
    int flip = 0;
    const int64_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    A s = 0;
    for (int64_t c = threadIdx.x; c < cols; c += 1024) s += to_acc(xr[c]);
    const A inv_n = A(1) / A(cols);
    const A mean = group_sum<1024>(s, red, flip) * inv_n;
    A q = 0;
    for (int64_t c = threadIdx.x; c < cols; c += 1024) {
        const A d = to_acc(xr[c]) - mean;
        q += d * d;
    }
    const A rstd = rsqrt_acc(group_sum<1024>(q, red, flip) * inv_n + eps);
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

// Walks rows blockIdx.x * RPB + group, + gridDim.x * RPB, ...; partial[blockIdx.x] = {sums of dy z, sums of dy}.
template <typename T, int VEC, int TPR, int NV>
__global__ void __launch_bounds__(TPR > LN_BLOCK ? TPR : LN_BLOCK)
ln_backward_kernel(int64_t rows, int cols, const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                   const T* __restrict__ scale, const typename AccOf<T>::type* __restrict__ mean,
                   const typename AccOf<T>::type* __restrict__ rstd, T* __restrict__ dx, int64_t lddx,
                   typename AccOf<T>::type* __restrict__ partial) {
    using A = typename AccOf<T>::type;
    using P = Pack<T, VEC>;
    constexpr int BLOCK = TPR > LN_BLOCK ? TPR : LN_BLOCK;
    constexpr int RPB = BLOCK / TPR;
    __shared__ Two<A> red[64];
    int flip = 0;
    const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
    const int c0 = t * VEC;
    P sc[NV];
    A acc_s[NV][VEC], acc_o[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = c0 + i * TPR * VEC;
        if (scale && c < cols) sc[i] = *reinterpret_cast<const P*>(scale + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) { acc_s[i][e] = 0; acc_o[i][e] = 0; }
    }
    const A inv_n = A(1) / A(cols);
    const int64_t step = int64_t(gridDim.x) * RPB;
    P bx[NV], bg[NV];
    A mu = 0, r = 0;
    auto fetch = [&](int64_t row) {
        if (row >= rows) return;
        mu = mean[row];
        r = rstd[row];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = c0 + i * TPR * VEC;
            if (c < cols) {
                bx[i] = *reinterpret_cast<const P*>(x + row * ldx + c);
                bg[i] = *reinterpret_cast<const P*>(dy + row * lddy + c);
            }
        }
    };
    fetch(int64_t(blockIdx.x) * RPB + grp);
    // every group of the block makes the same number of turns: the sums of wide rows meet at barriers
    for (int64_t base = int64_t(blockIdx.x) * RPB; base < rows; base += step) {
        const int64_t row = base + grp;
        const bool live = row < rows;
        P cx[NV], cg[NV];
        const A cmu = mu, cr = r;
        A s1 = 0, s2 = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) { cx[i] = bx[i]; cg[i] = bg[i]; }
        fetch(row + step);                // the next row is on its way while this one is summed
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (c0 + i * TPR * VEC < cols && live) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const A z = (to_acc(cx[i].v[e]) - cmu) * cr, d = to_acc(cg[i].v[e]);
                    acc_s[i][e] += d * z;
                    acc_o[i][e] += d;
                    const A g = scale ? d * to_acc(sc[i].v[e]) : d;
                    s1 += g;
                    s2 += g * z;
                }
            }
        const Two<A> m = group_sum2<TPR>(s1, s2, red, flip);
        const A m1 = m.a * inv_n, m2 = m.b * inv_n;
        if (live) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = c0 + i * TPR * VEC;
                if (c < cols) {
                    P o;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const A z = (to_acc(cx[i].v[e]) - cmu) * cr, d = to_acc(cg[i].v[e]);
                        const A g = scale ? d * to_acc(sc[i].v[e]) : d;
                        o.v[e] = from_acc<T, A>(cr * (g - m1 - z * m2));
                    }
                    *reinterpret_cast<P*>(dx + row * lddx + c) = o;
                }
            }
        }
    }
    if (!partial) return;
    A* ps = partial + int64_t(blockIdx.x) * 2 * cols;
    if constexpr (RPB == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = c0 + i * TPR * VEC;
            if (c < cols) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) { ps[c + e] = acc_s[i][e]; ps[cols + c + e] = acc_o[i][e]; }
            }
        }
    } else {
        // the groups' sums, added in group order; a slice of columns at a time keeps the buffer small
        __shared__ A buf[RPB][TPR * VEC];
#pragma unroll
        for (int k = 0; k < 2 * NV; ++k) {
            const int i = k >> 1;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < VEC; ++e) buf[grp][c0 + e] = (k & 1) ? acc_o[i][e] : acc_s[i][e];
            __syncthreads();
            for (int j = threadIdx.x; j < TPR * VEC; j += BLOCK) {
                const int c = j + i * TPR * VEC;
                if (c < cols) {
                    A s = 0;
                    for (int g = 0; g < RPB; ++g) s += buf[g][j];
                    ps[(k & 1) * int64_t(cols) + c] = s;
                }
            }
        }
    }
}

// dscale / doffset: partial rows added in order, 32 columns per block, the rows over 8 warps.
template <typename T>
__global__ void __launch_bounds__(256)
ln_reduce_kernel(int n_parts, int64_t cols, const typename AccOf<T>::type* __restrict__ partial, T* __restrict__ dscale,
                 T* __restrict__ doffset) {
    using A = typename AccOf<T>::type;
    __shared__ A buf[8][33];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t c = int64_t(blockIdx.x) * 32 + lane;      // 0 .. 2 * cols
    A s = 0;
    if (c < 2 * cols)
#pragma unroll 4
        for (int p = warp; p < n_parts; p += 8) s += partial[int64_t(p) * 2 * cols + c];
    buf[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < 2 * cols) {
#pragma unroll
        for (int w = 1; w < 8; ++w) s += buf[w][lane];
        T* out = c < cols ? dscale : doffset;
        if (out) out[c < cols ? c : c - cols] = from_acc<T, A>(s);
    }
}

// Wide rows, backward: dx by one block per row; the weights' partial sums by a kernel over columns and row slices.
template <typename T>
__global__ void __launch_bounds__(1024)
ln_backward_wide_kernel(int64_t cols, const T* __restrict__ dy, int64_t lddy, const T* __restrict__ x, int64_t ldx,
                        const T* __restrict__ scale, const typename AccOf<T>::type* __restrict__ mean,
                        const typename AccOf<T>::type* __restrict__ rstd, T* __restrict__ dx, int64_t lddx) {
    using A = typename AccOf<T>::type;
    __shared__ Two<A> red[64];
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
    const Two<A> m = group_sum2<1024>(s1, s2, red, flip);
    const A m1 = m.a / A(cols), m2 = m.b / A(cols);
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

// The group of threads a row is given: the smallest that holds it.  Wider groups than needed leave lanes idle on
// narrow rows; more elements per thread than these cost the registers that keep rows in flight.
//   16-byte accesses: up to 4 per thread.  Rows whose width or alignment rules them out are read element by element,
//   up to 8 per thread in groups of a warp or less and 16 in larger ones.
struct LnArgs {
    cudaStream_t st;
    int64_t rows, cols;
    const void *dy, *x, *scale, *offset;
    int64_t lddy, ldx, ldo;
    double eps;
    void *out, *mean, *rstd;
    void* partial;
    int grid;               // backward: blocks
};

int sm_count() {
    static int n[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    if (n[dev] == 0) {
        int v = 0;
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1) v = 148;
        n[dev] = v;
    }
    return n[dev];
}

template <typename T, int VEC, int TPR, int NV>
void run_forward(const LnArgs& a) {
    using A = typename AccOf<T>::type;
    constexpr int BLOCK = TPR > LN_BLOCK ? TPR : LN_BLOCK;
    constexpr int RPB = BLOCK / TPR;
    ln_forward_kernel<T, VEC, TPR, NV><<<unsigned(ceil_div(a.rows, RPB)), BLOCK, 0, a.st>>>(
        a.rows, int(a.cols), static_cast<const T*>(a.x), a.ldx, static_cast<const T*>(a.scale),
        static_cast<const T*>(a.offset), A(a.eps), static_cast<T*>(a.out), a.ldo, static_cast<A*>(a.mean),
        static_cast<A*>(a.rstd));
}

template <typename T, int VEC, int TPR, int NV>
void run_backward(const LnArgs& a) {
    using A = typename AccOf<T>::type;
    constexpr int BLOCK = TPR > LN_BLOCK ? TPR : LN_BLOCK;
    ln_backward_kernel<T, VEC, TPR, NV><<<unsigned(a.grid), BLOCK, 0, a.st>>>(
        a.rows, int(a.cols), static_cast<const T*>(a.dy), a.lddy, static_cast<const T*>(a.x), a.ldx,
        static_cast<const T*>(a.scale), static_cast<const A*>(a.mean), static_cast<const A*>(a.rstd),
        static_cast<T*>(a.out), a.ldo, static_cast<A*>(a.partial));
}

template <int VEC_, int TPR_, int NV_>
struct LnVariant {
    static constexpr int VEC = VEC_, TPR = TPR_, NV = NV_;
};

// Calls f(LnVariant<VEC, TPR, NV>{}) for the variant of `cols`; false for rows wider than a block holds.
template <typename T, typename F>
bool ln_variant(int64_t cols, bool vec, F&& f) {
    constexpr int V = 16 / sizeof(T);
    if (vec) {
        if (cols <= 8 * 4 * V) f(LnVariant<V, 8, 4>{});
        else if (cols <= 32 * 4 * V) f(LnVariant<V, 32, 4>{});
        else if (cols <= 128 * 4 * V) f(LnVariant<V, 128, 4>{});
        else if (cols <= 512 * 4 * V) f(LnVariant<V, 512, 4>{});
        else return false;
    } else {
        if (cols <= 8 * 8) f(LnVariant<1, 8, 8>{});
        else if (cols <= 32 * 8) f(LnVariant<1, 32, 8>{});
        else if (cols <= 128 * 16) f(LnVariant<1, 128, 16>{});
        else if (cols <= 512 * 16) f(LnVariant<1, 512, 16>{});
        else return false;
    }
    return true;
}

template <typename T>
bool aligned_rows(int64_t cols, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> lds) {
    constexpr int64_t V = 16 / sizeof(T);
    if (cols % V) return false;
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) % 16) return false;
    for (int64_t l : lds)
        if (l % V) return false;
    return true;
}

template <typename T>
int ln_forward_t(const LnArgs& a) {
    using A = typename AccOf<T>::type;
    const bool vec = aligned_rows<T>(a.cols, {a.x, a.scale, a.offset, a.out}, {a.ldx, a.ldo});
    const bool done = ln_variant<T>(a.cols, vec, [&](auto v) { run_forward<T, decltype(v)::VEC, decltype(v)::TPR, decltype(v)::NV>(a); });
    if (!done)
        ln_forward_wide_kernel<T><<<unsigned(a.rows), 1024, 0, a.st>>>(
            a.cols, static_cast<const T*>(a.x), a.ldx, static_cast<const T*>(a.scale), static_cast<const T*>(a.offset),
            A(a.eps), static_cast<T*>(a.out), a.ldo, static_cast<A*>(a.mean), static_cast<A*>(a.rstd));
    NNVB_CUDA(cudaGetLastError());
    return NNVB_OK;
}

constexpr int LN_MAX_PARTS = 1024;

template <typename T>
int ln_backward_t(LnArgs a, void* dscale, void* doffset) {
    using A = typename AccOf<T>::type;
    const bool vec = aligned_rows<T>(a.cols, {a.dy, a.x, a.scale, a.out}, {a.lddy, a.ldx, a.ldo});
    const int sms = sm_count();
    const bool done = ln_variant<T>(a.cols, vec, [&](auto v) {
        constexpr int TPR = decltype(v)::TPR, BLOCK = TPR > LN_BLOCK ? TPR : LN_BLOCK;
        const int64_t per_sm = BLOCK > 256 ? 2 : 4;
        a.grid = int(std::min<int64_t>({ceil_div(a.rows, BLOCK / TPR), sms * per_sm, LN_MAX_PARTS}));
        run_backward<T, decltype(v)::VEC, decltype(v)::TPR, decltype(v)::NV>(a);
    });
    if (!done) {
        ln_backward_wide_kernel<T><<<unsigned(a.rows), 1024, 0, a.st>>>(
            a.cols, static_cast<const T*>(a.dy), a.lddy, static_cast<const T*>(a.x), a.ldx, static_cast<const T*>(a.scale),
            static_cast<const A*>(a.mean), static_cast<const A*>(a.rstd), static_cast<T*>(a.out), a.ldo);
        if (a.partial) {
            NNVB_CUDA(cudaGetLastError());
            const int64_t cb = ceil_div(a.cols, 256);
            a.grid = int(std::max<int64_t>(1, std::min<int64_t>({a.rows, LN_MAX_PARTS, ceil_div(int64_t(sms) * 8, cb)})));
            ln_weights_wide_kernel<T><<<dim3(unsigned(cb), unsigned(a.grid)), 256, 0, a.st>>>(
                a.rows, a.cols, static_cast<const T*>(a.dy), a.lddy, static_cast<const T*>(a.x), a.ldx,
                static_cast<const A*>(a.mean), static_cast<const A*>(a.rstd), static_cast<A*>(a.partial));
        }
    }
    NNVB_CUDA(cudaGetLastError());
    if (a.partial) {
        ln_reduce_kernel<T><<<unsigned(ceil_div(2 * a.cols, 32)), 256, 0, a.st>>>(
            a.grid, a.cols, static_cast<const A*>(a.partial), static_cast<T*>(dscale), static_cast<T*>(doffset));
        NNVB_CUDA(cudaGetLastError());
    }
    return NNVB_OK;
}

}  // namespace

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

extern "C" {

int nnvb_layer_norm_forward(void* stream, int dtype, int64_t rows, int64_t cols, const void* x, int64_t ldx,
                            const void* scale, const void* offset, double eps, void* y, int64_t ldy, void* mean,
                            void* rstd) {
    NNVB_REQUIRE(dtype_bytes(dtype) > 0, "nnvb_layer_norm_forward: unknown element type %d", dtype);
    NNVB_REQUIRE(rows >= 0 && cols >= 1 && rows < (int64_t(1) << 31) && cols < (int64_t(1) << 31),
                 "nnvb_layer_norm_forward: bad sizes (rows=%lld, cols=%lld)", (long long)rows, (long long)cols);
    NNVB_REQUIRE(ldx >= cols && ldy >= cols, "nnvb_layer_norm_forward: rows overlap (cols=%lld, ldx=%lld, ldy=%lld)",
                 (long long)cols, (long long)ldx, (long long)ldy);
    NNVB_REQUIRE(eps >= 0 && eps < 1e30, "nnvb_layer_norm_forward: eps must be finite and not negative");
    if (rows == 0) return NNVB_OK;
    NNVB_REQUIRE(x && y, "nnvb_layer_norm_forward: NULL pointer");
    LnArgs a{static_cast<cudaStream_t>(stream), rows, cols, nullptr, x, scale, offset, 0, ldx, ldy, eps, y, mean, rstd,
             nullptr, 0};
    switch (dtype) {
        case NNVB_F64: return ln_forward_t<double>(a);
        case NNVB_F32: return ln_forward_t<float>(a);
        case NNVB_BF16: return ln_forward_t<__nv_bfloat16>(a);
        default: return ln_forward_t<__half>(a);
    }
}

int64_t nnvb_layer_norm_workspace(int dtype, int64_t rows, int64_t cols) {
    if (dtype_bytes(dtype) == 0 || rows < 0 || cols < 1) return 0;
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
    const bool weights = dscale || doffset;
    if (weights) {
        NNVB_REQUIRE(workspace && workspace_bytes >= nnvb_layer_norm_workspace(dtype, rows, cols) &&
                         reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                     "nnvb_layer_norm_backward: the weights' gradients need a 16-byte aligned workspace of %lld bytes",
                     (long long)nnvb_layer_norm_workspace(dtype, rows, cols));
    }
    LnArgs a{st, rows, cols, dy, x, scale, nullptr, lddy, ldx, lddx, 0.0, dx, const_cast<void*>(mean),
             const_cast<void*>(rstd), weights ? workspace : nullptr, 0};
    switch (dtype) {
        case NNVB_F64: return ln_backward_t<double>(a, dscale, doffset);
        case NNVB_F32: return ln_backward_t<float>(a, dscale, doffset);
        case NNVB_BF16: return ln_backward_t<__nv_bfloat16>(a, dscale, doffset);
        default: return ln_backward_t<__half>(a, dscale, doffset);
    }
}

}  // extern "C"
