// Attention over an encoder's states on the tensor cores: bf16 and fp16 tensors with head sizes up to 128 whose rows
// TMA can read (16-byte aligned, sizes a multiple of 8).
//
// Forward.  A block of twelve warps takes 256 positions of one head as two tiles of 128 rows and walks over the states in
// tiles of 128.  Warp 9 copies Q once and the K and V tiles through a ring of shared-memory stages (TMA); warp 8
// issues the products: S = Q K^T into tensor memory, then O += P V with P read from tensor memory and O kept there.
// Warps 0-3 and 4-7 hold one row of a tile per thread: read S, take the row's maximum, write P = exp2(c S - c m) over
// S as 16-bit values, and add the row's sum.  The two tiles alternate: while one is in its softmax the other's
// products run, so the tensor pipe sees S and P V of one tile during the exponentials of the other.
//
// Where such blocks are few, a cluster of up to 16 shares the states of one and joins its rows in distributed shared
// memory.
//
// The running maximum m is raised lazily: O is only rescaled when a row's maximum has grown by more than a factor of
// 2^8 over the m in use, so weights stay below 2^8, which 16-bit P and fp32 sums hold without loss; after the first
// tiles the rescale is rare.  P is rounded to the tensors' type because the product takes 16-bit operands; its
// row sum is added in fp32 before the rounding.  fp16 P carries a factor 2^7, up to the type's end: without it weights
// below 2^-14 lose bits, which shows where one state outweighs the others and its V does not matter.
//
// At long lengths the tensor pipe and shared memory need 1024 cycles each for a tile of states (Q K^T reads 8 KB for each 64
// cycles of the pipe, all that shared memory delivers), and each is busy 0.61 of the time while all SMs have blocks; the
// rest goes to the hand-overs between products and exponentials.  8 x 2048 x 4096 x 16 x 128 bf16: 525 us, 1.05 PFLOP/s.
//
// A block takes an SM's registers whole (the backward kernels 55 of 64 K), so no other block of this kind waits for its
// tensor memory while it waits for the rest of its cluster.
//
// Every wait is bounded (about 0.2 s): a block whose hand-over breaks stops issuing, waits for its own copies and products
// to end, frees its tensor memory and writes its rows as NaN.
#include <cooperative_groups.h>

#include <mutex>

#include "attention.cuh"
#include "tcgen05.cuh"

namespace cg = cooperative_groups;

namespace nnvb {
namespace {

constexpr int ROWS = 128;                          // rows of a tile of positions, states of a tile
constexpr int FWD_THREADS = 384;
constexpr int EMULATED = 4;                        // of 16 exponentials run on the FMA pipe (0: 44.7 us, 2: 43.5, 4: 42.7,
                                                   // 6: 45.9 at 8 x 1024 x 1024 x 8 x 128; within 2 % of one another
                                                   // at 8 x 2048 x 4096 x 16 x 128)

template <typename T> constexpr bool is_bf16 = false;
template <> constexpr bool is_bf16<__nv_bfloat16> = true;

// two values as the 16-bit halves of a register, the first in the low half
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    __nv_bfloat162 x = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&x);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    __half2 x = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&x);
}

// the halves of a packed register as floats
template <typename T> __device__ __forceinline__ float unpack_lo(uint32_t x);
template <typename T> __device__ __forceinline__ float unpack_hi(uint32_t x);
template <> __device__ __forceinline__ float unpack_lo<__nv_bfloat16>(uint32_t x) { return __uint_as_float(x << 16); }
template <> __device__ __forceinline__ float unpack_hi<__nv_bfloat16>(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
template <> __device__ __forceinline__ float unpack_lo<__half>(uint32_t x) { return __half2float(__ushort_as_half(x & 0xffff)); }
template <> __device__ __forceinline__ float unpack_hi<__half>(uint32_t x) { return __half2float(__ushort_as_half(x >> 16)); }

// 2^x to about 2 units in the last place, 0 below 2^-126: the weights' own rounding is 2^15 times coarser
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// 2^x on the FMA pipe, for a share of the weights: the exponential unit takes 16 a cycle, half of what the tensor pipe
// needs of them.  x = i + f with f in [-1/2, 1/2]; 2^f by the polynomial of degree 4 that interpolates it at the
// Chebyshev points (relative error below 5e-6, a 500th of P's rounding), times 2^i.  x <= 15 here.  From -126.5 down, -inf
// included, i is -127, whose bits as a float's exponent are those of 0: the same flush to zero as ex2's.
__device__ __forceinline__ Pair<float> ex2_poly(Pair<float> x) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-127.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-127.f));
    const float magic = 12582912.f;                    // 1.5 * 2^23: adding it rounds to an integer in the low bits
    const Pair<float> r = add2(x, both(magic));
    const Pair<float> f = add2(x, mul2(add2(r, both(-magic)), both(-1.f)));
    Pair<float> y = both(9.666368515e-03f);
    y = fma2(y, f, both(5.592197584e-02f));
    y = fma2(y, f, both(2.402234904e-01f));
    y = fma2(y, f, both(6.931210452e-01f));
    y = fma2(y, f, both(1.000000000e+00f));
    // as a product, not as a sum of bits: NaN stays NaN
    return mul2(y, {__int_as_float((__float_as_int(r.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(r.y) << 23) + 0x3f800000)});
}

// eight results, one rounding each
template <typename T>
__device__ __forceinline__ void store8(T* to, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(to) = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}

struct TcMaps {
    CUtensorMap q, k, v;
};

// Rows of positions are those of 2^gs query heads that share a state head, heads of a position side by side: few positions
// of grouped heads fill tiles, and K and V are read once for them.  A map's dimensions are channel, head, token, batch
// entry; a broadcast dimension is stored as one entry.
__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* m, int boxes, int box_bytes, int token, int head, int batch,
                                          uint64_t* bar) {
    for (int i = 0; i < boxes; ++i) tma_load_4d(static_cast<char*>(dst) + i * box_bytes, m, i * 64, head, token, batch, bar);
}

template <int DP>
struct FwdSmem {
    static constexpr int BOX = ROWS * 128;                 // 64 elements x 128 rows
    static constexpr int TILE = BOX * (DP / 64);
    static constexpr int STAGES = DP == 128 ? 4 : 8;
    static constexpr int BYTES = TILE * (2 + STAGES) + 1024;
};

template <typename T, int DP>
__global__ void __launch_bounds__(FWD_THREADS, 1)
attn_fwd_tc_kernel(const __grid_constant__ TcMaps maps, AttnArgs a, int gs) {
    using SM = FwdSmem<DP>;
    constexpr int STAGES = SM::STAGES;
    extern __shared__ unsigned char raw[];
    unsigned char* base = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
    unsigned char* sq = base;
    unsigned char* ring = base + 2 * SM::TILE;
    __shared__ uint64_t full[STAGES], empty[STAGES], q_full, s_ready[2], p_ready[2][2], o_ready[2], tail, drain;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ float row_m[2 * ROWS], row_l[2 * ROWS];             // clusters

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), world = int(cluster.num_blocks());
    const int rows = a.Lq << gs, groups = a.Hq >> gs, in_group = (1 << gs) - 1;
    const int tiles = (rows + 2 * ROWS - 1) / (2 * ROWS);
    const int unit = int(blockIdx.x) / world;
    const int q0 = unit % tiles * 2 * ROWS;
    const int h = (unit / tiles % groups) << gs, b = unit / tiles / groups;      // h: the group's first head
    const int g = h / (a.Hq / a.Hkv);
    const int n = attn_len(a, b);
    const int live = rows - q0 > ROWS ? 2 : 1;             // tiles of rows this block holds
    auto out_at = [&](int row) {
        return static_cast<T*>(const_cast<void*>(a.o)) + int64_t(b) * a.os[0] + int64_t(row >> gs) * a.os[1] +
               int64_t(h + (row & in_group)) * a.os[2];
    };
    auto lse_at = [&](int row) {
        return static_cast<float*>(a.lse) + (int64_t(b) * a.Hq + h + (row & in_group)) * a.Lq + (row >> gs);
    };
    // tiles of states: every world-th is this block's
    const int all_steps = (n + ROWS - 1) / ROWS, steps = all_steps > rank ? (all_steps - rank + world - 1) / world : 0;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        mbar_init(&q_full, 1);
        mbar_init(&tail, 1);
        mbar_init(&drain, 1);
        for (int t = 0; t < 2; ++t) {
            mbar_init(&s_ready[t], 1);
            mbar_init(&o_ready[t], 1);
            for (int half = 0; half < 2; ++half) mbar_init(&p_ready[t][half], 4);
        }
        mbar_init_fence();
    }
    if (warp == 8) tmem_alloc(&tmem_slot, 512);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    constexpr uint32_t tmem = 0;           // all 512 columns are this block's, so they start at column 0
    volatile int* abort = &abort_flag;

    // 384 threads at 168 registers = 256 at 208 + 128 at 88: a softmax thread holds a row of 128 scores (8 x 2048 x 4096 x
    // 16 x 128: with 168 registers 9 % slower and the scores read twice, 5 % slower with them spilled)
    if (warp >= 8) {
        setmaxnreg_dec<88>();
        if (warp == 9) {
            // ---- copies -------------------------------------------------------------------------------------------
            const int kb = a.ks[0] ? b : 0, kh = a.ks[2] ? g : 0, vb = a.vs[0] ? b : 0, vh = a.vs[2] ? g : 0;
            if (lane == 0 && steps > 0) {
                mbar_expect_bytes(&q_full, uint32_t(live) * SM::TILE);
                for (int t = 0; t < live; ++t)
                    load_tile(sq + t * SM::TILE, &maps.q, DP / 64, SM::BOX, (q0 + t * ROWS) >> gs, a.qs[2] ? h : 0, a.qs[0] ? b : 0, &q_full);
            }
            int it = 0;
            bool ok = true, cleared = false;
            for (int i = 0; i < steps && ok; ++i) {
                for (int kv = 0; kv < 2; ++kv, ++it) {
                    const int s = it % STAGES;
                    if (it >= STAGES) ok = mbar_wait_fast(&empty[s], (it / STAGES - 1) & 1, abort);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    unsigned char* dst = ring + s * SM::TILE;
                    const int row = (rank + i * world) * ROWS, rest = n - row;
                    // V rows behind the valid states may hold anything, and 0 * NaN is NaN: they are cleared here.  (K needs
                    // nothing: its rows only make scores that are masked.)
                    if (kv == 1 && rest < ROWS && n < a.Lk) {
                        if (lane == 0) {
                            mbar_expect_bytes(&tail, SM::TILE);
                            load_tile(dst, &maps.v, DP / 64, SM::BOX, row, vh, vb, &tail);
                        }
                        cleared = true;
                        ok = __all_sync(0xffffffffu, mbar_wait_fast(&tail, 0, abort));
                        for (int j = lane; j < (ROWS - rest) * 8 * (DP / 64); j += 32) {
                            const int box = j / ((ROWS - rest) * 8), r = j % ((ROWS - rest) * 8);
                            *reinterpret_cast<uint4*>(dst + box * SM::BOX + rest * 128 + r * 16) = make_uint4(0, 0, 0, 0);
                        }
                        async_proxy_fence();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&full[s]);
                    } else if (lane == 0) {
                        mbar_expect_bytes(&full[s], SM::TILE);
                        load_tile(dst, kv ? &maps.v : &maps.k, DP / 64, SM::BOX, row, kv ? vh : kh, kv ? vb : kb, &full[s]);
                    }
                }
            }
            // A block does not leave while a copy writes to its memory.  The products have waited for all of them, unless some
            // warp gave up.
            if (lane == 0 && steps > 0) {
                mbar_wait(&q_full, 0, 1 << 20);
                if (cleared) mbar_wait(&tail, 0, 1 << 20);
                for (int j = it > STAGES ? it - STAGES : 0; j < it; ++j) mbar_wait(&full[j % STAGES], (j / STAGES) & 1, 1 << 20);
            }
            __syncwarp();
        } else if (warp == 8) {
            // ---- products -----------------------------------------------------------------------------------------
            const uint32_t leader = elect_lane();
            if (steps > 0) {
                constexpr uint32_t id_s = mma_idesc(is_bf16<T>, 128, ROWS, false);
                constexpr uint32_t id_o = mma_idesc(is_bf16<T>, 128, DP, true);
                const int ksteps = (a.D + 15) / 16;
                const uint32_t q_addr = smem_u32(sq), r_addr = smem_u32(ring);
                auto scores = [&](int t, int s) {
                    const uint32_t qd = desc_k_major(q_addr + t * SM::TILE), kd = desc_k_major(r_addr + s * SM::TILE);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k) {
                        const uint32_t off = ((k / 4) * SM::BOX + (k % 4) * 32) >> 4;
                        if (k < ksteps) mma_ss(leader, tmem + t * 128, qd + off, kd + off, id_s, k > 0);
                    }
                    mma_commit(leader, &s_ready[t]);
                };
                bool ok = warp_wait(&q_full, 0, abort) && warp_wait(&full[0], 0, abort);
                if (ok) {
                    for (int t = 0; t < live; ++t) scores(t, 0);
                    mma_commit(leader, &empty[0]);
                }
                for (int i = 0; i < steps && ok; ++i) {
                    const int vi = 2 * i + 1, ki = 2 * i + 2;
                    const bool next = i + 1 < steps;
                    ok = warp_wait(&full[vi % STAGES], (vi / STAGES) & 1, abort);
                    if (ok && next) ok = warp_wait(&full[ki % STAGES], (ki / STAGES) & 1, abort);
                    for (int t = 0; t < live && ok; ++t) {
                        const uint32_t vd = desc_mn_major(r_addr + (vi % STAGES) * SM::TILE, SM::BOX);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {         // the first half runs while the second's exponentials do
                            ok = ok && warp_wait(&p_ready[t][half], i & 1, abort);
                            if (!ok) break;
                            tmem_fence_after();
#pragma unroll
                            for (int k = half * ROWS / 32; k < (half + 1) * ROWS / 32; ++k)
                                mma_ts(leader, tmem + 256 + t * 128, tmem + t * 128 + k * 8, vd + k * (2048 >> 4), id_o, i > 0 || k > 0);
                        }
                        if (!ok) break;
                        // S of the next states goes over P of these: products issued by one thread run in order
                        if (next) scores(t, ki % STAGES);
                        else mma_commit(leader, &o_ready[t]);
                    }
                    if (ok) {
                        mma_commit(leader, &empty[vi % STAGES]);
                        if (next) mma_commit(leader, &empty[ki % STAGES]);
                    }
                }
                // the last commit has arrived: nothing touches this block's barriers after it has left
                if (ok) ok = warp_wait(&empty[(2 * steps - 1) % STAGES], ((2 * steps - 1) / STAGES) & 1, abort);
                if (!ok) {                     // gave up: nothing may still write to the tensor memory that is freed below
                    mma_commit(leader, &drain);
                    mbar_wait(&drain, 0, 1 << 20);
                }
            }
            __syncwarp();
        }
    } else {
        setmaxnreg_inc<208>();
        if (warp / 4 < live) {
            // ---- softmax: one row per thread ------------------------------------------------------------------------
            const int t = warp / 4;
            const uint32_t lanes = tmem + (uint32_t(warp % 4) << 21);
            const uint32_t s_at = lanes + t * 128, o_at = lanes + 256 + t * 128;
            const int row = q0 + t * ROWS + (warp % 4) * 32 + lane;
            const float c = float(a.scale * LOG2E);
            // m: the maximum in use, of the scores without the factor; fp16: less 7 powers of two, except where scores are so
            // large (2^20) that the rounding of m c would take P past the type's end
            const float below = fminf(7.f / c, 3e38f), large = 1048576.f / c;
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int i = 0; i < steps; ++i) {
                ok = mbar_wait_fast(&s_ready[t], i & 1, abort);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tmem_fence_after();
                const int rest = n - (rank + i * world) * ROWS;
                uint32_t s[4][32];
#pragma unroll
                for (int j = 0; j < 4; ++j) tmem_load32(s[j], s_at + j * 32);
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    tmem_wait_load(s[j]);
                    if (rest < (j + 1) * 32) {
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (j * 32 + e >= rest) s[j][e] = 0xff800000u;        // -inf
                    }
#pragma unroll
                    for (int e = 0; e < 32; e += 2) mx[e / 2 % 4] = max3(mx[e / 2 % 4], __uint_as_float(s[j][e]), __uint_as_float(s[j][e + 1]));
                }
                float top = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]);
                if (!is_bf16<T> && fabsf(top) < large) top -= below;
                const bool raise = m == -INFINITY ? top > m : (top - m) * c > 8.f;
                if (i == 0) {
                    m = top;
                } else if (__any_sync(0xffffffffu, raise)) {
                    const float f = raise ? (m == -INFINITY ? 0.f : ex2((m - top) * c)) : 1.f;
                    if (raise) m = top;
                    l *= f;
#pragma unroll 1
                    for (int j = 0; j < DP / 32; ++j) {
                        uint32_t o[32];
                        tmem_load32(o, o_at + j * 32);
                        tmem_wait_load(o);
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                        tmem_store32(o_at + j * 32, o);
                    }
                }
                const float mc = m == -INFINITY ? 0.f : m * c;
                Pair<float> sum[2] = {both(0.f), both(0.f)};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t p[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        Pair<float> x = fma2({__uint_as_float(s[j][e]), __uint_as_float(s[j][e + 1])}, both(c), both(-mc));
                        x = e % 16 < EMULATED ? ex2_poly(x) : Pair<float>{ex2(x.x), ex2(x.y)};
                        sum[e / 2 % 2] = add2(sum[e / 2 % 2], x);
                        p[e / 2] = pack2<T>(x.x, x.y);
                    }
                    // over columns 16 j .. 16 j + 15 of S, which have been read by now
                    tmem_store16(s_at + j * 16, p);
                    if (j % 2) {
                        tmem_wait_store();
                        tmem_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_ready[t][j / 2]);    // one arrival a warp: arrivals on a barrier are served one by one
                    }
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            if (ok && steps > 0) {
                ok = mbar_wait_fast(&o_ready[t], 0, abort);
                // a cluster's results go over the ring, which the other tile's products read too
                if (world > 1 && live > 1) ok = ok && mbar_wait_fast(&o_ready[1 - t], 0, abort);
                ok = __all_sync(0xffffffffu, ok);
            }
            tmem_fence_after();
            if (world > 1) {
                const int r = t * ROWS + (warp % 4) * 32 + lane;
                if (!ok) l = NAN;
                row_m[r] = m;
                row_l[r] = l;
                float4* mine = reinterpret_cast<float4*>(ring) + r * (DP / 4);
#pragma unroll 1
                for (int j = 0; j < DP / 32; ++j) {
                    uint32_t o[32];
                    if (steps > 0) {
                        tmem_load32(o, o_at + j * 32);
                        tmem_wait_load(o);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (steps > 0)
                            x = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]),
                                            __uint_as_float(o[4 * e + 3]));
                        mine[(j * 8 + e + r) % (DP / 4)] = x;          // rows turned against each other: one bank a lane
                    }
                }
            } else {
                const float f = !ok ? NAN : (n > 0 ? 1.f / l : 0.f);
                T* out = out_at(row);
#pragma unroll 1
                for (int j = 0; j < DP / 32; ++j) {
                    uint32_t o[32];
                    if (n > 0 && ok) {
                        tmem_load32(o, o_at + j * 32);
                        tmem_wait_load(o);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0;
                    }
                    if (row < rows) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            if (j * 32 + e < a.D) {
                                float x[8];
#pragma unroll
                                for (int u = 0; u < 8; ++u) x[u] = __uint_as_float(o[e + u]) * f;
                                store8<T>(out + j * 32 + e, x);
                            }
                        }
                    }
                }
                if (a.lse && row < rows)
                    *lse_at(row) = !ok ? NAN : (n > 0 ? m * float(a.scale) + logf(l) : -INFINITY);
            }
        }
    }
    if (world > 1) {
        // the blocks of a cluster hold the same rows over different states: each writes a share of the rows, added in
        // block order
        cluster.sync();
        const float c = float(a.scale * LOG2E);
        for (int i = rank * FWD_THREADS + threadIdx.x; i < live * ROWS * (DP / 8); i += world * FWD_THREADS) {
            const int r = i / (DP / 8), d = i % (DP / 8) * 8, row = q0 + r;
            if (row >= rows) continue;
            float top = -INFINITY, sum = 0.f, x[8] = {};
            for (int w = 0; w < world; ++w) top = fmaxf(top, *cluster.map_shared_rank(&row_m[r], w));
            const float base = top == -INFINITY ? 0.f : top;
            for (int w = 0; w < world; ++w) {
                const float f = ex2((*cluster.map_shared_rank(&row_m[r], w) - base) * c);
                sum += *cluster.map_shared_rank(&row_l[r], w) * f;
                const float4* part = cluster.map_shared_rank(reinterpret_cast<float4*>(ring), w) + r * (DP / 4);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float4 y = part[(d / 4 + u + r) % (DP / 4)];
                    x[u * 4] += y.x * f; x[u * 4 + 1] += y.y * f; x[u * 4 + 2] += y.z * f; x[u * 4 + 3] += y.w * f;
                }
            }
            const float f = n > 0 ? 1.f / sum : 0.f;
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] *= f;
            if (d < a.D) store8<T>(out_at(row) + d, x);
            if (d == 0 && a.lse) *lse_at(row) = n > 0 ? top * float(a.scale) + logf(sum) : -INFINITY;
        }
        cluster.sync();                    // nobody leaves while its shared memory is read
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 8) tmem_free(tmem, 512);
}

// ---------------------------------------------------------------------------
// Backward.  P = exp2(c S - lse'), dS = P (dP - delta) with lse' = lse log2 e.  One kernel serves both passes:
//   dQ       resident Q and dO (128 positions), streamed K and V:   S = Q K^T,  dP = dO V^T,  dQ += dS K,  W += P K
//   dK, dV   resident K and V (128 states), streamed Q and dO of every query head of the group:
//            S^T = K Q^T,  dP^T = V dO^T,  dV += P^T dO,  dK += dS^T Q
// so each gradient row is summed in tensor memory by one block, in a fixed order.  Separate passes compute S and dP
// twice: eight products a pair instead of the five of one pass that would add to dQ atomically, ten with the second terms of
// dS.  A streamed tile of 64 rows of 128 channels takes 1280 cycles of the tensor pipe and moves 176 KB through shared memory,
// 1375 cycles; the pipe is busy 0.60 of the time in both passes.  4 x 2048 x 2048 x 16 x 128 bf16: 650 us, 0.53 PFLOP/s
// counted as five products, 1.06 as the ten that run.
//
// Streamed tiles have 64 rows, which lets two of them be in flight in tensor memory beside 128 x 128 accumulators;
// they serve as K-major operand of S and dP and as MN-major operand of the gradients.  Sixteen warps do the softmax
// arithmetic: two warpgroups per tile in flight, one row and half of its 64 columns per thread (with one warpgroup per
// tile the products waited for it: a quarter of the tensor pipe's cycles were used).
//
// fp16 holds 2^-24 to 65504, dS anything from the product of two small gradients up to |dP| of large ones: it is lifted by a
// power of two that its bound |dS| <= 2 max |dO_i| max |v_j| (Euclidean norms, P <= 1) puts below 2^15, and the gradient is
// divided by it again.  With two terms that leaves 2^-40 of the bound.  dQ takes the norm of 16 of its rows of dO, dK of all.
//
// Roundings: P is rounded to the tensors' type, as in the forward pass.  dS enters its product as the sum of two
// 16-bit values (its rounding and the rounding of what is left): its rounding error would be as large as that of storing dQ
// and dK, and the terms of dS cancel in their row sums.  delta comes from the
// stored output (delta0), and where a row's weight lies on a few states its rounding is larger than dP - delta: the error
// of dq would be 7.2e-3 instead of 1.7e-3 for bf16 queries of 16 sigma over 129 states.  So the dQ pass sums what dS with
// delta0 misses, e = sum_j P (dP - delta0), takes it back as dQ - e W at its end and leaves delta0 + e for the
// other pass.  P's rounding enters e W in second order only.

constexpr int BROWS = 64;                          // rows of a streamed tile
constexpr int BWD_SOFT = 512;                      // threads of the softmax arithmetic
constexpr int BWD_THREADS = BWD_SOFT + 64;

template <int DP>
struct BwdSmem {
    static constexpr int ABOX = ROWS * 128, ATILE = ABOX * (DP / 64);
    static constexpr int BBOX = BROWS * 128, BTILE = BBOX * (DP / 64);
    static constexpr int STATS = 2 * BROWS * 4;    // lse' and delta of the streamed positions
    static constexpr int STAGES = 4;
    static constexpr int BYTES = 2 * ATILE + STAGES * 2 * BTILE + STAGES * STATS + 1024;
};

struct BwdMaps {
    CUtensorMap a0, a1, b0, b1;
};

// The largest of a block's 16 values, which 16 lanes each hold.
__device__ __forceinline__ void block_largest(float s, float* to) {
    __shared__ float part[8];
    s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, 16, 32));
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) s = fmaxf(s, part[w]);
        *to = s;
    }
}

// fp16 loses bits below 2^-14: weights enter their products times 2^12.
template <typename T> constexpr float P_SHIFT = is_bf16<T> ? 0.f : 12.f;

// stats: [B, groups of heads, RowsP] lse' (less P_SHIFT) then the same of delta, a group's rows rounded up to 64: those behind hold +inf and 0.
// fp16: then the largest squared norm of dO of every 16 rows, and of V of every V_CHUNK states (blocks from row_blocks on).
template <typename T>
__global__ void __launch_bounds__(256)
attn_stats_tc_kernel(AttnArgs a, int RowsP, int gs, unsigned row_blocks) {
    const int lane = threadIdx.x % 16;
    const int groups = a.Hq >> gs;
    const int64_t count = int64_t(a.B) * groups * RowsP;
    if (!is_bf16<T> && blockIdx.x >= row_blocks) {
        const int chunks = (a.Lk + V_CHUNK - 1) / V_CHUNK, at = int(blockIdx.x - row_blocks);
        const int j0 = at % chunks * V_CHUNK + threadIdx.x / 16, g = at / chunks % a.Hkv, b = at / chunks / a.Hkv, n = attn_len(a, b);
        const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + g * a.vs[2] + lane * 8;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < V_CHUNK / 16; ++i) {
            const int j = j0 + 16 * i;
            float x = 0.f;
            if (j < n && lane * 8 < a.D) {
                const auto y = *reinterpret_cast<const Pack<T, 8>*>(v + j * a.vs[1]);
#pragma unroll
                for (int e = 0; e < 8; ++e) x += to_acc(y.v[e]) * to_acc(y.v[e]);
            }
            for (int w = 8; w > 0; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w, 32);
            s = fmaxf(s, x);
        }
        block_largest(s, static_cast<float*>(a.delta) + 2 * count + count / 16 + at);
        return;
    }
    const int64_t i = int64_t(blockIdx.x) * 16 + threadIdx.x / 16;
    const int row = int(i % RowsP), b = int(i / RowsP / groups);
    const int h = (int(i / RowsP % groups) << gs) + (row & ((1 << gs) - 1)), r = row >> gs;
    const bool live = i < count && r < a.Lq;
    float s = 0.f, norm = 0.f;
    if (live && lane * 8 < a.D) {
        const auto o = *reinterpret_cast<const Pack<T, 8>*>(static_cast<const T*>(a.o) + b * a.os[0] + r * a.os[1] + h * a.os[2] + lane * 8);
        const auto d = *reinterpret_cast<const Pack<T, 8>*>(static_cast<const T*>(a.dout) + b * a.dos[0] + r * a.dos[1] + h * a.dos[2] + lane * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s += to_acc(o.v[e]) * to_acc(d.v[e]);
            norm += to_acc(d.v[e]) * to_acc(d.v[e]);
        }
    }
    for (int w = 8; w > 0; w >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, w, 32);
        if (!is_bf16<T>) norm += __shfl_xor_sync(0xffffffffu, norm, w, 32);
    }
    if (!is_bf16<T>) block_largest(norm, static_cast<float*>(a.delta) + 2 * count + blockIdx.x);
    if (i < count && lane == 0) {
        float* st = static_cast<float*>(a.delta);
        st[i] = live ? static_cast<const float*>(a.lse)[(int64_t(b) * a.Hq + h) * a.Lq + r] * float(LOG2E) - P_SHIFT<T> : INFINITY;
        st[count + i] = s;
    }
}

// The power of two that lifts values of at most `bound` to below 2^15, and its inverse.
__device__ __forceinline__ void ds_factor(float bound, float* up, float* down) {
    if (!(bound > 0.f && bound < INFINITY)) return;          // nothing to lift, or results that are not finite anyway
    const int e = (__float_as_int(bound) >> 23) - 127;       // a bound of fp16 norms: 2^-48 .. 2^42
    *up = __int_as_float((127 + 14 - e) << 23);
    *down = __int_as_float((127 - 14 + e) << 23);
}

template <typename T, int DP, bool KV>
__global__ void __launch_bounds__(BWD_THREADS, 1)
attn_bwd_tc_kernel(const __grid_constant__ BwdMaps maps, AttnArgs a, int RowsP, int gs) {
    using SM = BwdSmem<DP>;
    constexpr int STAGES = SM::STAGES;
    constexpr bool SCALED = !is_bf16<T>;
    extern __shared__ unsigned char raw[];
    unsigned char* base = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
    unsigned char* res = base;                             // A0, A1
    unsigned char* ring = base + 2 * SM::ATILE;            // B0, B1 per stage
    float* stats = reinterpret_cast<float*>(ring + STAGES * 2 * SM::BTILE);
    __shared__ uint64_t full[STAGES], empty[STAGES], a_full, s_ready[2], p_ready[2], o_ready, tail, drain;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    __shared__ float row_sum[4][ROWS], row_miss[ROWS];
    __shared__ float factor;

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    // rows and heads (dQ: groups of 2^gs) of this pass
    const int rows = a.Lq << gs, groups = a.Hq >> gs;
    const int own_len = KV ? a.Lk : rows, own_heads = KV ? a.Hkv : groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), world = int(cluster.num_blocks());
    const int tiles = (own_len + ROWS - 1) / ROWS;
    const int unit = int(blockIdx.x) / world;
    const int r0 = unit % tiles * ROWS;
    const int oh = unit / tiles % own_heads, b = unit / tiles / own_heads;
    const int G = (a.Hq / a.Hkv) >> gs;                    // groups that share a state head
    const int n = attn_len(a, b);
    // streamed tiles: rows of the groups that share the state head, or valid states
    const int per_head = KV ? (rows + BROWS - 1) / BROWS : (n + BROWS - 1) / BROWS;
    const int all_steps = KV ? (r0 < n ? per_head * G : 0) : per_head;
    // every world-th is this block's
    const int steps = all_steps > rank ? (all_steps - rank + world - 1) / world : 0;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        mbar_init(&a_full, 1);
        mbar_init(&o_ready, 1);
        mbar_init(&tail, 1);
        mbar_init(&drain, 1);
        for (int t = 0; t < 2; ++t) { mbar_init(&s_ready[t], 1); mbar_init(&p_ready[t], 8); }
        mbar_init_fence();
    }
    if (warp == 16) tmem_alloc(&tmem_slot, 512);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    constexpr uint32_t tmem = 0;           // all 512 columns are this block's, so they start at column 0
    volatile int* abort = &abort_flag;
    constexpr float P_SCALE = is_bf16<T> ? 1.f : 4096.f;           // 2^P_SHIFT
    // Tensor memory, columns: tile in flight t at 128 t: S 0..63, dP 64..127; the accumulators of dQ / dK at 256 and of
    // W / dV at 384.  The two warpgroups of a tile own 32 columns of S and of dP each and put their 16-bit operands there:
    // P over the lower half of their columns of S, the rest of dS over the upper half, dS over the lower half of dP.
    const float* st_lse = static_cast<const float*>(a.delta);
    float* st_delta = static_cast<float*>(a.delta) + int64_t(a.B) * groups * RowsP;
    // where row r of a gradient begins
    auto grad_at = [&](int r) {
        return KV ? ((int64_t(b) * a.Lk + r) * a.Hkv + oh) * a.D
                  : ((int64_t(b) * a.Lq + (r >> gs)) * a.Hq + (oh << gs) + (r & ((1 << gs) - 1))) * a.D;
    };

    if (warp == 17) {
        // ---- copies -------------------------------------------------------------------------------------------
        const int64_t *as0 = KV ? a.ks : a.qs, *as1 = KV ? a.vs : a.dos, *bs0 = KV ? a.qs : a.ks, *bs1 = KV ? a.dos : a.vs;
        if (lane == 0 && steps > 0) {
            mbar_expect_bytes(&a_full, 2 * SM::ATILE);
            const int ah = KV ? oh : oh << gs, token = KV ? r0 : r0 >> gs;
            load_tile(res, &maps.a0, DP / 64, SM::ABOX, token, as0[2] ? ah : 0, as0[0] ? b : 0, &a_full);
            load_tile(res + SM::ATILE, &maps.a1, DP / 64, SM::ABOX, token, as1[2] ? ah : 0, as1[0] ? b : 0, &a_full);
        }
        int it = 0;
        bool ok = true, cleared = false;
        for (; it < steps && ok; ++it) {
            const int s = it % STAGES;
            if (it >= STAGES) ok = mbar_wait_fast(&empty[s], (it / STAGES - 1) & 1, abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int at_step = rank + it * world;
            const int sh = KV ? oh * G + at_step / per_head : oh / G;      // streamed group or state head
            const int bh = KV ? sh << gs : sh;
            const int row = at_step % per_head * BROWS;
            unsigned char* dst = ring + s * 2 * SM::BTILE;
            const int rest = KV ? BROWS : n - row;
            // K rows behind the valid states may hold anything, and 0 * NaN is NaN: they are cleared here.  (V
            // needs nothing: its rows only make columns of dP that are masked.)
            const bool clear = !KV && rest < BROWS && n < a.Lk;
            uint64_t* bar = clear ? &tail : &full[s];
            if (lane == 0) {
                mbar_expect_bytes(bar, 2 * SM::BTILE + (KV ? SM::STATS : 0));
                const int token = KV ? row >> gs : row;
                load_tile(dst, &maps.b0, DP / 64, SM::BBOX, token, bs0[2] ? bh : 0, bs0[0] ? b : 0, bar);
                load_tile(dst + SM::BTILE, &maps.b1, DP / 64, SM::BBOX, token, bs1[2] ? bh : 0, bs1[0] ? b : 0, bar);
                if (KV) {
                    const int64_t at = (int64_t(b) * groups + sh) * RowsP + row;
                    bulk_copy_g2s(stats + s * 2 * BROWS, st_lse + at, BROWS * 4, bar);
                    bulk_copy_g2s(stats + s * 2 * BROWS + BROWS, st_delta + at, BROWS * 4, bar);
                }
            }
            if (clear) {
                cleared = true;
                ok = __all_sync(0xffffffffu, mbar_wait_fast(&tail, 0, abort));
                const int pieces = (BROWS - rest) * 8;
                for (int j = lane; j < pieces * (DP / 64); j += 32) {
                    const int box = j / pieces, r = j % pieces;
                    *reinterpret_cast<uint4*>(dst + box * SM::BBOX + rest * 128 + r * 16) = make_uint4(0, 0, 0, 0);
                }
                async_proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[s]);
            }
        }
        if (lane == 0 && steps > 0) {      // a block does not leave while a copy writes to its memory
            mbar_wait(&a_full, 0, 1 << 20);
            if (cleared) mbar_wait(&tail, 0, 1 << 20);
            for (int j = it > STAGES ? it - STAGES : 0; j < it; ++j) mbar_wait(&full[j % STAGES], (j / STAGES) & 1, 1 << 20);
        }
        __syncwarp();
    } else if (warp == 16) {
        // ---- products -----------------------------------------------------------------------------------------
        const uint32_t leader = elect_lane();
        if (steps > 0) {
            constexpr uint32_t id_s = mma_idesc(is_bf16<T>, 128, BROWS, false);
            constexpr uint32_t id_g = mma_idesc(is_bf16<T>, 128, DP, true);
            const int ksteps = (a.D + 15) / 16;
            const uint32_t a_addr = smem_u32(res), r_addr = smem_u32(ring);
            auto scores = [&](int j) {
                const uint32_t d = tmem + (j & 1) * 128, b_addr = r_addr + (j % STAGES) * 2 * SM::BTILE;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint32_t ad = desc_k_major(a_addr + w * SM::ATILE), bd = desc_k_major(b_addr + w * SM::BTILE);
#pragma unroll
                    for (int k = 0; k < DP / 16; ++k)
                        if (k < ksteps)
                            mma_ss(leader, d + w * 64, ad + (((k / 4) * SM::ABOX + (k % 4) * 32) >> 4), bd + (((k / 4) * SM::BBOX + (k % 4) * 32) >> 4),
                                   id_s, k > 0);
                }
                mma_commit(leader, &s_ready[j & 1]);
            };
            bool ok = warp_wait(&a_full, 0, abort) && warp_wait(&full[0], 0, abort);
            if (ok) scores(0);
            for (int j = 0; j < steps && ok; ++j) {
                if (j + 1 < steps) {
                    ok = warp_wait(&full[(j + 1) % STAGES], ((j + 1) / STAGES) & 1, abort);
                    // goes over P and dS of tile j - 1, whose products were issued before: they run in order
                    if (ok) scores(j + 1);
                }
                ok = ok && warp_wait(&p_ready[j & 1], (j / 2) & 1, abort);
                if (!ok) break;
                tmem_fence_after();
                const uint32_t d = tmem + (j & 1) * 128, b_addr = r_addr + (j % STAGES) * 2 * SM::BTILE;
                const uint32_t b0 = desc_mn_major(b_addr, SM::BBOX), b1 = desc_mn_major(b_addr + SM::BTILE, SM::BBOX);
#pragma unroll
                for (int k = 0; k < BROWS / 16; ++k) {
                    const uint32_t at = d + (k / 2) * 32 + (k % 2) * 8;
                    mma_ts(leader, tmem + 256, at + 64, b0 + k * (2048 >> 4), id_g, j > 0 || k > 0);
                    mma_ts(leader, tmem + 256, at + 16, b0 + k * (2048 >> 4), id_g, true);
                    mma_ts(leader, tmem + 384, at, (KV ? b1 : b0) + k * (2048 >> 4), id_g, j > 0 || k > 0);
                }
                mma_commit(leader, &empty[j % STAGES]);
            }
            if (ok) {
                mma_commit(leader, &o_ready);
                ok = warp_wait(&o_ready, 0, abort);
            }
            if (!ok) {                     // gave up: nothing may still write to the tensor memory that is freed below
                mma_commit(leader, &drain);
                mbar_wait(&drain, 0, 1 << 20);
            }
        }
        __syncwarp();
    } else {
        // ---- P and dS ---------------------------------------------------------------------------------------------
        const int wg = warp / 4, t = wg / 2, half = wg % 2;
        const uint32_t lanes = tmem + (uint32_t(warp % 4) << 21);
        const uint32_t s_at = lanes + t * 128 + half * 32, d_at = s_at + 64;
        const int local = (warp % 4) * 32 + lane, row = r0 + local;
        const float c = float(a.scale * LOG2E);
        float my_lse = 0.f, my_delta = 0.f;
        const int64_t my_at = (int64_t(b) * groups + oh) * RowsP + row;
        if (!KV && row < rows) {
            my_lse = st_lse[my_at];
            my_delta = st_delta[my_at];
        }
        // fp16: what dS (beside P's 2^P_SHIFT) is multiplied with and divided by; the dQ pass leaves delta times dK's factor
        float up = 1.f, down = 1.f, head_up = 1.f;
        if (SCALED && all_steps > 0) {
            const int sh = KV ? oh : oh / G;
            const int64_t chunks = (a.Lk + V_CHUNK - 1) / V_CHUNK, row_chunks = int64_t(G) * (RowsP / 16);
            const float* of_rows = st_delta + int64_t(a.B) * groups * RowsP;
            const float* of_states = of_rows + int64_t(a.B) * a.Hkv * row_chunks + (int64_t(b) * a.Hkv + sh) * chunks;
            float v = 0.f, d = 0.f;
            for (int i = lane; i < (n + V_CHUNK - 1) / V_CHUNK; i += 32) v = fmaxf(v, of_states[i]);
            for (int64_t i = lane; i < row_chunks; i += 32) d = fmaxf(d, of_rows[(int64_t(b) * a.Hkv + sh) * row_chunks + i]);
            for (int w = 16; w > 0; w >>= 1) {
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, w, 32));
                d = fmaxf(d, __shfl_xor_sync(0xffffffffu, d, w, 32));
            }
            ds_factor(2.f * sqrtf(v * d), &up, &down);
            head_up = up *= 1.f / P_SCALE;
            if (!KV) {
                up = down = 1.f;
                if (row < rows) ds_factor(2.f * sqrtf(v * of_rows[my_at / 16]), &up, &down);
                up *= 1.f / P_SCALE;
            }
        }
        if (threadIdx.x == 0) factor = head_up;
        const float up_delta = up * my_delta;
        Pair<float> miss = both(0.f);
        bool ok = true;
        for (int j = t; j < steps; j += 2) {
            ok = mbar_wait_fast(&full[j % STAGES], (j / STAGES) & 1, abort) &&
                 mbar_wait_fast(&s_ready[t], (j / 2) & 1, abort);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tmem_fence_after();
            const float* sl = stats + (j % STAGES) * 2 * BROWS + half * 32;
            const int rest = KV ? 32 : n - (rank + j * world) * BROWS - half * 32;          // columns with weight
            uint32_t s[32];
            tmem_load32(s, s_at);
            tmem_wait_load(s);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                const Pair<float> lse = KV ? *reinterpret_cast<const Pair<float>*>(sl + e) : both(my_lse);
                const Pair<float> x = fma2({__uint_as_float(s[e]), __uint_as_float(s[e + 1])}, both(c), {-lse.x, -lse.y});
                s[e] = __float_as_uint(ex2(x.x));
                s[e + 1] = __float_as_uint(ex2(x.y));
            }
            if (!KV && rest < 32) {                        // the last tile: S and dP may hold anything there
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (e >= rest) s[e] = 0;
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                uint32_t d[16], p[8], hi[8], lo[8];
                tmem_load16(d, d_at + g * 16);
                tmem_wait_load(d);
                if (!KV && rest < 32) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (g * 16 + e >= rest) d[e] = 0;
                }
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const int col = g * 16 + e;
                    const Pair<float> pv{__uint_as_float(s[col]), __uint_as_float(s[col + 1])};
                    const Pair<float> dp{__uint_as_float(d[e]), __uint_as_float(d[e + 1])};
                    // dl: fp16: delta times the factor
                    const Pair<float> dl = KV ? *reinterpret_cast<const Pair<float>*>(sl + BROWS + col) : both(up_delta);
                    Pair<float> ds = mul2(pv, SCALED ? fma2(dp, both(up), Pair<float>{-dl.x, -dl.y}) : add2(dp, Pair<float>{-dl.x, -dl.y}));
                    if (!KV) miss = add2(miss, ds);
                    p[e / 2] = pack2<T>(pv.x, pv.y);
                    hi[e / 2] = pack2<T>(ds.x, ds.y);
                    ds = add2(ds, Pair<float>{-unpack_lo<T>(hi[e / 2]), -unpack_hi<T>(hi[e / 2])});
                    lo[e / 2] = pack2<T>(ds.x, ds.y);
                }
                tmem_store8(s_at + g * 8, p);
                tmem_store8(s_at + 16 + g * 8, lo);
                tmem_store8(d_at + g * 8, hi);
            }
            tmem_wait_store();
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[t]);           // one arrival a warp: arrivals on a barrier are served one by one
        }
        if (ok && steps > 0) ok = __all_sync(0xffffffffu, mbar_wait_fast(&o_ready, 0, abort));
        tmem_fence_after();
        float e = 0.f;                                     // dQ: what delta0 misses
        if (!KV) {
            row_sum[wg][local] = ok ? (miss.x + miss.y) * down : NAN;
            named_bar_sync(1, BWD_SOFT);
            e = (row_sum[0][local] + row_sum[1][local]) + (row_sum[2][local] + row_sum[3][local]);
            if (wg == 0) row_miss[local] = e;
            if (wg == 0 && world == 1 && row < rows) st_delta[my_at] = (my_delta + e) * head_up;
        }
        // dK: warpgroups 0 and 1, dV: 2 and 3, half of the columns each; dQ: every warpgroup a chunk of 32
        const bool value = KV && t == 1;
        const bool dead = KV && row >= n;                  // states without weight: their rows of S may hold anything
        const bool zero = ok && (steps == 0 || dead);
        const float fw = float(a.scale) / P_SCALE;
        const float f = !ok ? NAN : (value ? 1.f / P_SCALE : float(a.scale) * down);
        T* out = static_cast<T*>(KV ? (value ? a.dv : a.dk) : a.dq) + grad_at(row);
        const uint32_t o_at = lanes + 256 + (value ? 128 : 0);
        float4* mine = reinterpret_cast<float4*>(base) + ((value ? ROWS : 0) + local) * (DP / 4);
        constexpr int NJ = DP / 32;
        const int j0 = KV ? half * (NJ / 2) : wg, j1 = KV ? j0 + NJ / 2 : (wg < NJ ? wg + 1 : wg);
#pragma unroll 1
        for (int j = j0; j < j1; ++j) {
            uint32_t o[32];
            if (steps > 0 && ok) {
                tmem_load32(o, o_at + j * 32);
                tmem_wait_load(o);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(zero ? 0.f : (ok ? __uint_as_float(o[i]) * f : NAN));
            if (!KV) {
                uint32_t w[32];
                if (steps > 0 && ok) {
                    tmem_load32(w, o_at + 128 + j * 32);
                    tmem_wait_load(w);
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float x = zero ? 0.f : (ok ? __uint_as_float(w[i]) * fw : NAN);
                    if (world > 1) w[i] = __float_as_uint(x);
                    else o[i] = __float_as_uint(__uint_as_float(o[i]) - e * x);
                }
                if (world > 1)
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        (mine + ROWS * (DP / 4))[(j * 8 + i + local) % (DP / 4)] = *reinterpret_cast<const float4*>(w + 4 * i);
            }
            if (world > 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i) mine[(j * 8 + i + local) % (DP / 4)] = *reinterpret_cast<const float4*>(o + 4 * i);
            } else if (row < own_len) {
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    if (j * 32 + i < a.D) {
                        float x[8];
#pragma unroll
                        for (int u = 0; u < 8; ++u) x[u] = __uint_as_float(o[i + u]);
                        store8<T>(out + j * 32 + i, x);
                    }
                }
            }
        }
    }
    if (world > 1) {
        // the blocks' sums over their streamed tiles, added in block order; each writes a share of the rows
        cluster.sync();
        constexpr int PARTS = KV ? 2 : 1;
        auto joined = [&](float (&x)[8], int pr, int d) {
            for (int w = 0; w < world; ++w) {
                const float4* part = cluster.map_shared_rank(reinterpret_cast<float4*>(base), w) + pr * (DP / 4);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float4 y = part[(d / 4 + u + pr) % (DP / 4)];
                    x[u * 4] += y.x; x[u * 4 + 1] += y.y; x[u * 4 + 2] += y.z; x[u * 4 + 3] += y.w;
                }
            }
        };
        for (int i = rank * BWD_THREADS + threadIdx.x; i < PARTS * ROWS * (DP / 8); i += world * BWD_THREADS) {
            const int pr = i / (DP / 8), r = pr % ROWS, d = i % (DP / 8) * 8, row = r0 + r;
            if (row >= own_len || d >= a.D) continue;
            float x[8] = {};
            joined(x, pr, d);
            if (!KV) {
                float w[8] = {}, e = 0.f;
                joined(w, ROWS + r, d);
                for (int k = 0; k < world; ++k) e += *cluster.map_shared_rank(&row_miss[r], k);
#pragma unroll
                for (int u = 0; u < 8; ++u) x[u] -= e * w[u];
                float* delta = st_delta + (int64_t(b) * groups + oh) * RowsP + row;
                if (d == 0) *delta = (*delta + e) * factor;
            }
            store8<T>(static_cast<T*>(KV ? (pr >= ROWS ? a.dv : a.dk) : a.dq) + grad_at(row) + d, x);
        }
        cluster.sync();                    // nobody leaves while its shared memory is read
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 16) tmem_free(tmem, 512);
}

// ---------------------------------------------------------------------------
// host side

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
    static std::once_flag once;
    static EncodeFn fn = nullptr;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) == cudaSuccess && r == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(p);
    });
    return fn;
}

// Boxes of 64 elements x 2^gs heads x `rows` / 2^gs tokens; a dimension with stride 0 (broadcast, or of one entry) has one entry.
int make_map(CUtensorMap* m, int dtype, const void* p, const int64_t (&s)[3], int64_t D, int64_t tokens, int64_t heads,
             int64_t batch, int rows, int gs) {
    EncodeFn fn = encode_fn();
    if (!fn) {
        set_error("nnvb_cross_attention: the CUDA driver does not offer cuTensorMapEncodeTiled");
        return NNVB_E_CUDA;
    }
    const cuuint64_t dims[4] = {cuuint64_t(D), cuuint64_t(s[2] ? heads : 1), cuuint64_t(tokens), cuuint64_t(s[0] ? batch : 1)};
    auto stride = [](int64_t e) { return cuuint64_t(e ? e * 2 : 16); };
    const cuuint64_t strides[3] = {stride(s[2]), stride(s[1]), stride(s[0])};
    const cuuint32_t box[4] = {64, cuuint32_t(1) << gs, cuuint32_t(rows >> gs), 1}, one[4] = {1, 1, 1, 1};
    const CUresult r = fn(m, dtype == NNVB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                          const_cast<void*>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("nnvb_cross_attention: cuTensorMapEncodeTiled failed (%d)", int(r));
        return NNVB_E_CUDA;
    }
    return NNVB_OK;
}

// Heads of a group whose positions are packed into rows: the largest power of two that divides the group, at most a
// streamed tile's 64 rows; tensors whose heads are broadcast are not packed.
int pack_shift(const AttnArgs& a, bool backward) {
    int gs = 0;
    if (a.qs[2] == 0 || (backward && a.dos[2] == 0)) return 0;
    while (gs < 6 && (a.Hq / a.Hkv) % (2 << gs) == 0) ++gs;
    return gs;
}

// rows TMA can read: 16-byte aligned, strides a multiple of 16 bytes below 2^40; tokens must not be broadcast
bool tma_rows(const void* p, const int64_t (&s)[3], int64_t tokens) {
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
    for (int64_t x : s)
        if (x % 8 || x >= (int64_t(1) << 39)) return false;
    return tokens <= 1 || s[1] > 0;
}

// Launches `units` blocks, or clusters of up to 16 where blocks are few and walk over many tiles (`steps`).
template <typename K, typename... Args>
int launch_shared(K kernel, int64_t units, int64_t steps, int threads, int smem, cudaStream_t st, Args... args) {
    const int sms = sm_count();
    int world = 1;
    const int most = units <= 4 ? 16 : 8;              // a GPC has room for one cluster of 16 such blocks
    while (world < most && units * world * 2 <= sms && world * 4 <= steps) world *= 2;
    NNVB_REQUIRE(units * world < (int64_t(1) << 31), "nnvb_cross_attention: too many tiles (%lld) for one launch", (long long)units);
    NNVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (world > 8) NNVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(units * world));
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = size_t(smem);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = unsigned(world);
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    NNVB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return NNVB_OK;
}

template <typename T, int DP>
int forward_t(cudaStream_t st, const AttnArgs& a) {
    using SM = FwdSmem<DP>;
    TcMaps maps{};
    const int gs = pack_shift(a, false);
    NNVB_TRY(make_map(&maps.q, a.dtype, a.q, a.qs, a.D, a.Lq, a.Hq, a.B, ROWS, gs));
    if (a.Lk > 0) {
        NNVB_TRY(make_map(&maps.k, a.dtype, a.k, a.ks, a.D, a.Lk, a.Hkv, a.B, ROWS, 0));
        NNVB_TRY(make_map(&maps.v, a.dtype, a.v, a.vs, a.D, a.Lk, a.Hkv, a.B, ROWS, 0));
    }
    return launch_shared(attn_fwd_tc_kernel<T, DP>, ceil_div(int64_t(a.Lq) << gs, 2 * ROWS) * (a.Hq >> gs) * a.B,
                         ceil_div(a.Lk, ROWS), FWD_THREADS, SM::BYTES, st, maps, a, gs);
}

template <typename T, int DP>
int backward_t(cudaStream_t st, const AttnArgs& a) {
    using SM = BwdSmem<DP>;
    const int gs = pack_shift(a, true);
    const int64_t rows = int64_t(a.Lq) << gs, groups = a.Hq >> gs, RowsP = round_up(rows, BROWS);
    const int64_t count = RowsP * a.B * groups;
    const int64_t row_blocks = count / 16, blocks = row_blocks + (is_bf16<T> ? 0 : ceil_div(a.Lk, V_CHUNK) * a.Hkv * a.B);
    NNVB_REQUIRE(blocks < (int64_t(1) << 31), "nnvb_cross_attention_backward: too many rows (%lld)", (long long)blocks * 16);
    attn_stats_tc_kernel<T><<<unsigned(blocks), 256, 0, st>>>(a, int(RowsP), gs, unsigned(row_blocks));
    NNVB_CUDA(cudaGetLastError());
    BwdMaps mq{}, mk{};
    NNVB_TRY(make_map(&mq.a0, a.dtype, a.q, a.qs, a.D, a.Lq, a.Hq, a.B, ROWS, gs));
    NNVB_TRY(make_map(&mq.a1, a.dtype, a.dout, a.dos, a.D, a.Lq, a.Hq, a.B, ROWS, gs));
    NNVB_TRY(make_map(&mq.b0, a.dtype, a.k, a.ks, a.D, a.Lk, a.Hkv, a.B, BROWS, 0));
    NNVB_TRY(make_map(&mq.b1, a.dtype, a.v, a.vs, a.D, a.Lk, a.Hkv, a.B, BROWS, 0));
    NNVB_TRY(make_map(&mk.a0, a.dtype, a.k, a.ks, a.D, a.Lk, a.Hkv, a.B, ROWS, 0));
    NNVB_TRY(make_map(&mk.a1, a.dtype, a.v, a.vs, a.D, a.Lk, a.Hkv, a.B, ROWS, 0));
    NNVB_TRY(make_map(&mk.b0, a.dtype, a.q, a.qs, a.D, a.Lq, a.Hq, a.B, BROWS, gs));
    NNVB_TRY(make_map(&mk.b1, a.dtype, a.dout, a.dos, a.D, a.Lq, a.Hq, a.B, BROWS, gs));
    NNVB_TRY(launch_shared(attn_bwd_tc_kernel<T, DP, false>, ceil_div(rows, ROWS) * groups * a.B, ceil_div(a.Lk, BROWS), BWD_THREADS,
                           SM::BYTES, st, mq, a, int(RowsP), gs));
    return launch_shared(attn_bwd_tc_kernel<T, DP, true>, ceil_div(a.Lk, ROWS) * a.Hkv * a.B,
                         RowsP / BROWS * ((a.Hq / a.Hkv) >> gs), BWD_THREADS, SM::BYTES, st, mk, a, int(RowsP), gs);
}

}  // namespace

bool attn_tc_takes_forward(const AttnArgs& a) {
    if (a.dtype != NNVB_BF16 && a.dtype != NNVB_F16) return false;
    if (a.D > 128 || a.D % 8) return false;
    for (int64_t x : a.os)
        if (x % 8) return false;
    return reinterpret_cast<uintptr_t>(a.o) % 16 == 0 && tma_rows(a.q, a.qs, a.Lq) && tma_rows(a.k, a.ks, a.Lk) &&
           tma_rows(a.v, a.vs, a.Lk);
}

int attn_forward_tc(cudaStream_t st, const AttnArgs& a) {
    if (a.dtype == NNVB_BF16) return a.D <= 64 ? forward_t<__nv_bfloat16, 64>(st, a) : forward_t<__nv_bfloat16, 128>(st, a);
    return a.D <= 64 ? forward_t<__half, 64>(st, a) : forward_t<__half, 128>(st, a);
}

bool attn_tc_takes_backward(const AttnArgs& a) {
    auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    return attn_tc_takes_forward(a) && tma_rows(a.dout, a.dos, a.Lq) && aligned(a.dq) && aligned(a.dk) && aligned(a.dv);
}

int attn_backward_tc(cudaStream_t st, const AttnArgs& a) {
    if (a.dtype == NNVB_BF16) return a.D <= 64 ? backward_t<__nv_bfloat16, 64>(st, a) : backward_t<__nv_bfloat16, 128>(st, a);
    return a.D <= 64 ? backward_t<__half, 64>(st, a) : backward_t<__half, 128>(st, a);
}

}  // namespace nnvb
