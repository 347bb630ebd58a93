// Attention over an encoder's states on the tensor cores: bf16 and fp16 tensors with head sizes up to 128 whose rows
// TMA can read (16-byte aligned, sizes a multiple of 8).
//
// Forward.  A block of ten warps takes 256 positions of one head as two tiles of 128 rows and walks over the states in
// tiles of 128.  Warp 9 copies Q once and the K and V tiles through a ring of shared-memory stages (TMA); warp 8
// issues the products: S = Q K^T into tensor memory, then O += P V with P read from tensor memory and O kept there.
// Warps 0-3 and 4-7 hold one row of a tile per thread: read S, take the row's maximum, write P = exp2(c S - c m) over
// S as 16-bit values, and add the row's sum.  The two tiles alternate: while one is in its softmax the other's
// products run, so the tensor pipe sees S and P V of one tile during the exponentials of the other.
//
// The running maximum m is raised lazily: O is only rescaled when a row's maximum has grown by more than a factor of
// 2^8 over the m in use, so weights stay below 2^8, which 16-bit P and fp32 sums hold without loss; after the first
// tiles the rescale is rare.  P is rounded to the tensors' type because the product takes 16-bit operands; its
// row sum is added in fp32 before the rounding.
#include <mutex>

#include "attention.cuh"
#include "tcgen05.cuh"

namespace nnvb {
namespace {

__device__ unsigned long long g_timeouts;         // waits given up (a broken hand-over; the rows are written as NaN)

constexpr int ROWS = 128;                          // rows of a tile of positions, states of a tile
constexpr int FWD_THREADS = 320;

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

// 2^x to about 2 units in the last place, 0 below 2^-126: the weights' own rounding is 2^15 times coarser
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct TcMaps {
    CUtensorMap q, k, v, dout;
};

// coordinates of a head in a map; a broadcast dimension is stored as one entry
__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* m, int boxes, int box_bytes, int row, int head, int batch,
                                          uint64_t* bar) {
    for (int i = 0; i < boxes; ++i) tma_load_4d(static_cast<char*>(dst) + i * box_bytes, m, i * 64, row, head, batch, bar);
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
attn_fwd_tc_kernel(const __grid_constant__ TcMaps maps, AttnArgs a) {
    using SM = FwdSmem<DP>;
    constexpr int STAGES = SM::STAGES;
    extern __shared__ unsigned char raw[];
    unsigned char* base = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
    unsigned char* sq = base;
    unsigned char* ring = base + 2 * SM::TILE;
    __shared__ uint64_t full[STAGES], empty[STAGES], q_full, s_ready[2], p_ready[2], o_ready[2], tail, drain;
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int tiles = (a.Lq + 2 * ROWS - 1) / (2 * ROWS);
    const int q0 = int(blockIdx.x % tiles) * 2 * ROWS;
    const int h = int(blockIdx.x / tiles % a.Hq), b = int(blockIdx.x / tiles / a.Hq);
    const int g = h / (a.Hq / a.Hkv);
    const int n = attn_len(a, b);
    const int live = a.Lq - q0 > ROWS ? 2 : 1;             // tiles of positions this block holds
    const int steps = (n + ROWS - 1) / ROWS;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        mbar_init(&q_full, 1);
        mbar_init(&tail, 1);
        mbar_init(&drain, 1);
        for (int t = 0; t < 2; ++t) { mbar_init(&s_ready[t], 1); mbar_init(&p_ready[t], ROWS); mbar_init(&o_ready[t], 1); }
        mbar_init_fence();
    }
    if (warp == 8) tmem_alloc(&tmem_slot, 512);
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = tmem_slot;
    volatile int* abort = &abort_flag;

    if (warp == 9) {
        // ---- copies -------------------------------------------------------------------------------------------
        const int kb = a.ks[0] ? b : 0, kh = a.ks[2] ? g : 0, vb = a.vs[0] ? b : 0, vh = a.vs[2] ? g : 0;
        if (lane == 0 && n > 0) {
            mbar_expect_bytes(&q_full, uint32_t(live) * SM::TILE);
            for (int t = 0; t < live; ++t)
                load_tile(sq + t * SM::TILE, &maps.q, DP / 64, SM::BOX, q0 + t * ROWS, a.qs[2] ? h : 0, a.qs[0] ? b : 0, &q_full);
        }
        int it = 0;
        bool ok = true;
        for (int i = 0; i < steps && ok; ++i) {
            for (int kv = 0; kv < 2; ++kv, ++it) {
                const int s = it % STAGES;
                if (it >= STAGES) ok = mbar_wait_or_abort(&empty[s], (it / STAGES - 1) & 1, abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                unsigned char* dst = ring + s * SM::TILE;
                const int rest = n - i * ROWS;
                // V rows behind the valid states may hold anything, and 0 * NaN is NaN: they are cleared here.  (K needs
                // nothing: its rows only make scores that are masked.)
                if (kv == 1 && rest < ROWS && n < a.Lk) {
                    if (lane == 0) {
                        mbar_expect_bytes(&tail, SM::TILE);
                        load_tile(dst, &maps.v, DP / 64, SM::BOX, i * ROWS, vh, vb, &tail);
                    }
                    ok = __all_sync(0xffffffffu, mbar_wait_or_abort(&tail, 0, abort));
                    for (int j = lane; j < (ROWS - rest) * 8 * (DP / 64); j += 32) {
                        const int box = j / ((ROWS - rest) * 8), r = j % ((ROWS - rest) * 8);
                        *reinterpret_cast<uint4*>(dst + box * SM::BOX + rest * 128 + r * 16) = make_uint4(0, 0, 0, 0);
                    }
                    async_proxy_fence();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&full[s]);
                } else if (lane == 0) {
                    mbar_expect_bytes(&full[s], SM::TILE);
                    load_tile(dst, kv ? &maps.v : &maps.k, DP / 64, SM::BOX, i * ROWS, kv ? vh : kh, kv ? vb : kb, &full[s]);
                }
            }
        }
        if (!ok && lane == 0) {            // gave up: the copies issued so far still write to this block's memory
            if (n > 0) mbar_wait(&q_full, 0, 1 << 20);
            for (int j = it > STAGES ? it - STAGES : 0; j < it; ++j) mbar_wait(&full[j % STAGES], (j / STAGES) & 1, 1 << 20);
        }
    } else if (warp == 8) {
        // ---- products -----------------------------------------------------------------------------------------
        if (lane == 0 && n > 0) {
            constexpr uint32_t id_s = mma_idesc(is_bf16<T>, 128, ROWS, false);
            constexpr uint32_t id_o = mma_idesc(is_bf16<T>, 128, DP, true);
            const int ksteps = (a.D + 15) / 16;
            const uint32_t q_addr = smem_u32(sq), r_addr = smem_u32(ring);
            auto scores = [&](int t, int s) {
                for (int k = 0; k < ksteps; ++k) {
                    const uint32_t off = (k / 4) * SM::BOX + (k % 4) * 32;
                    mma_ss(tmem + t * 128, desc_k_major(q_addr + t * SM::TILE + off), desc_k_major(r_addr + s * SM::TILE + off), id_s, k > 0);
                }
                mma_commit(&s_ready[t]);
            };
            bool ok = mbar_wait_or_abort(&q_full, 0, abort) && mbar_wait_or_abort(&full[0], 0, abort);
            if (ok) {
                for (int t = 0; t < live; ++t) scores(t, 0);
                mma_commit(&empty[0]);
            }
            for (int i = 0; i < steps && ok; ++i) {
                const int vi = 2 * i + 1, ki = 2 * i + 2;
                const bool next = i + 1 < steps;
                ok = mbar_wait_or_abort(&full[vi % STAGES], (vi / STAGES) & 1, abort);
                if (ok && next) ok = mbar_wait_or_abort(&full[ki % STAGES], (ki / STAGES) & 1, abort);
                for (int t = 0; t < live && ok; ++t) {
                    ok = mbar_wait_or_abort(&p_ready[t], i & 1, abort);
                    if (!ok) break;
                    tmem_fence_after();
                    for (int k = 0; k < ROWS / 16; ++k)
                        mma_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8,
                               desc_mn_major(r_addr + (vi % STAGES) * SM::TILE + k * 2048, SM::BOX), id_o, i > 0 || k > 0);
                    // S of the next states goes over P of these: products issued by one thread run in order
                    if (next) scores(t, ki % STAGES);
                    else mma_commit(&o_ready[t]);
                }
                if (ok) {
                    mma_commit(&empty[vi % STAGES]);
                    if (next) mma_commit(&empty[ki % STAGES]);
                }
            }
            // the last commit has arrived: nothing touches this block's barriers after it has left
            if (ok) ok = mbar_wait_or_abort(&empty[(2 * steps - 1) % STAGES], ((2 * steps - 1) / STAGES) & 1, abort);
            if (!ok) {                     // gave up: nothing may still write to the tensor memory that is freed below
                mma_commit(&drain);
                mbar_wait(&drain, 0, 1 << 20);
            }
        }
        __syncwarp();
    } else if (warp / 4 < live) {
        // ---- softmax: one row per thread ------------------------------------------------------------------------
        const int t = warp / 4;
        const uint32_t lanes = tmem + (uint32_t(warp % 4) << 21);
        const uint32_t s_at = lanes + t * 128, o_at = lanes + 256 + t * 128;
        const int row = q0 + t * ROWS + (warp % 4) * 32 + lane;
        const float c = float(a.scale * LOG2E);
        float m = -INFINITY, l = 0.f;      // m: the maximum in use, of the scores without the factor
        bool ok = true;
        for (int i = 0; i < steps; ++i) {
            ok = mbar_wait_or_abort(&s_ready[t], i & 1, abort);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            tmem_fence_after();
            uint32_t s[4][32];
#pragma unroll
            for (int j = 0; j < 4; ++j) tmem_load32(s[j], s_at + j * 32);
            tmem_wait_load();
            const int rest = n - i * ROWS;
            if (rest < ROWS) {
#pragma unroll
                for (int j = 0; j < 128; ++j)
                    if (j >= rest) s[j / 32][j % 32] = 0xff800000u;        // -inf
            }
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 128; ++j) mx[j % 4] = fmaxf(mx[j % 4], __uint_as_float(s[j / 32][j % 32]));
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
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
                    tmem_wait_load();
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tmem_store32(o_at + j * 32, o);
                }
            }
            const float mc = m == -INFINITY ? 0.f : m * c;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                    const float x = ex2(__uint_as_float(s[j][e]) * c - mc), y = ex2(__uint_as_float(s[j][e + 1]) * c - mc);
                    sum[e / 2 % 4] += x;
                    sum[e / 2 % 4] += y;
                    p[e / 2] = pack2<T>(x, y);
                }
                tmem_store16(s_at + j * 16, p);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tmem_wait_store();
            tmem_fence_before();
            mbar_arrive(&p_ready[t]);
        }
        if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait_or_abort(&o_ready[t], 0, abort));
        tmem_fence_after();
        const float f = !ok ? NAN : (n > 0 ? 1.f / l : 0.f);
        T* out = static_cast<T*>(const_cast<void*>(a.o)) + int64_t(b) * a.os[0] + int64_t(row) * a.os[1] + int64_t(h) * a.os[2];
#pragma unroll 1
        for (int j = 0; j < DP / 32; ++j) {
            uint32_t o[32];
            if (n > 0 && ok) {
                tmem_load32(o, o_at + j * 32);
                tmem_wait_load();
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0;
            }
            if (row < a.Lq) {
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    if (j * 32 + e < a.D) {
                        uint4 w;
                        w.x = pack2<T>(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f);
                        w.y = pack2<T>(__uint_as_float(o[e + 2]) * f, __uint_as_float(o[e + 3]) * f);
                        w.z = pack2<T>(__uint_as_float(o[e + 4]) * f, __uint_as_float(o[e + 5]) * f);
                        w.w = pack2<T>(__uint_as_float(o[e + 6]) * f, __uint_as_float(o[e + 7]) * f);
                        *reinterpret_cast<uint4*>(out + j * 32 + e) = w;
                    }
                }
            }
        }
        if (a.lse && row < a.Lq)
            static_cast<float*>(a.lse)[(int64_t(b) * a.Hq + h) * a.Lq + row] =
                !ok ? NAN : (n > 0 ? m * float(a.scale) + logf(l) : -INFINITY);
    }
    tmem_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && abort_flag) atomicAdd(&g_timeouts, 1ull);
    if (warp == 8) tmem_free(tmem, 512);
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

// Boxes of 64 elements x `rows` tokens of one head; a dimension with stride 0 (broadcast, or of one entry) has one entry.
int make_map(CUtensorMap* m, int dtype, const void* p, const int64_t (&s)[3], int64_t D, int64_t tokens, int64_t heads,
             int64_t batch, int rows) {
    EncodeFn fn = encode_fn();
    if (!fn) {
        set_error("nnvb_cross_attention: the CUDA driver does not offer cuTensorMapEncodeTiled");
        return NNVB_E_CUDA;
    }
    const cuuint64_t dims[4] = {cuuint64_t(D), cuuint64_t(tokens), cuuint64_t(s[2] ? heads : 1), cuuint64_t(s[0] ? batch : 1)};
    auto stride = [](int64_t e) { return cuuint64_t(e ? e * 2 : 16); };
    const cuuint64_t strides[3] = {stride(s[1]), stride(s[2]), stride(s[0])};
    const cuuint32_t box[4] = {64, cuuint32_t(rows), 1, 1}, one[4] = {1, 1, 1, 1};
    const CUresult r = fn(m, dtype == NNVB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                          const_cast<void*>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("nnvb_cross_attention: cuTensorMapEncodeTiled failed (%d)", int(r));
        return NNVB_E_CUDA;
    }
    return NNVB_OK;
}

// rows TMA can read: 16-byte aligned, strides a multiple of 16 bytes below 2^40; tokens must not be broadcast
bool tma_rows(const void* p, const int64_t (&s)[3], int64_t tokens) {
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
    for (int64_t x : s)
        if (x % 8 || x >= (int64_t(1) << 39)) return false;
    return tokens <= 1 || s[1] > 0;
}

template <typename T, int DP>
int forward_t(cudaStream_t st, const AttnArgs& a) {
    using SM = FwdSmem<DP>;
    TcMaps maps{};
    NNVB_TRY(make_map(&maps.q, a.dtype, a.q, a.qs, a.D, a.Lq, a.Hq, a.B, ROWS));
    if (a.Lk > 0) {
        NNVB_TRY(make_map(&maps.k, a.dtype, a.k, a.ks, a.D, a.Lk, a.Hkv, a.B, ROWS));
        NNVB_TRY(make_map(&maps.v, a.dtype, a.v, a.vs, a.D, a.Lk, a.Hkv, a.B, ROWS));
    }
    const int64_t blocks = ceil_div(a.Lq, 2 * ROWS) * a.Hq * a.B;
    NNVB_REQUIRE(blocks < (int64_t(1) << 31), "nnvb_cross_attention: too many tiles (%lld) for one launch", (long long)blocks);
    auto kernel = attn_fwd_tc_kernel<T, DP>;
    NNVB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SM::BYTES));
    kernel<<<unsigned(blocks), FWD_THREADS, SM::BYTES, st>>>(maps, a);
    NNVB_CUDA(cudaGetLastError());
    return NNVB_OK;
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

}  // namespace nnvb
