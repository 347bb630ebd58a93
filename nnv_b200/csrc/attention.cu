// C entry points of the attention over an encoder's states: argument checks and the choice of kernel family.
#include <algorithm>
#include <cmath>

#include "attention.cuh"

using namespace nnvb;

namespace {

constexpr int64_t I31 = (int64_t(1) << 31) - 4096;      // sizes whose last tile still counts in 32 bits

int check_desc(const char* who, const nnvb_attention_desc* d) {
    NNVB_REQUIRE(d, "%s: NULL descriptor", who);
    NNVB_REQUIRE(dtype_bytes(d->dtype) > 0, "%s: unknown element type %d", who, d->dtype);
    NNVB_REQUIRE(d->batch >= 0 && d->q_len >= 0 && d->kv_len >= 0 && d->batch < I31 && d->q_len < I31 && d->kv_len < I31,
                 "%s: bad sizes (batch=%lld, q_len=%lld, kv_len=%lld)", who, (long long)d->batch, (long long)d->q_len,
                 (long long)d->kv_len);
    NNVB_REQUIRE(d->q_heads >= 1 && d->kv_heads >= 1 && d->q_heads < I31 && d->q_heads % d->kv_heads == 0,
                 "%s: %lld query heads over %lld state heads", who, (long long)d->q_heads, (long long)d->kv_heads);
    NNVB_REQUIRE(d->q_len * (d->q_heads / d->kv_heads) < I31, "%s: bad sizes (%lld positions of %lld heads a state head)", who,
                 (long long)d->q_len, (long long)(d->q_heads / d->kv_heads));
    NNVB_REQUIRE(d->head_dim >= 1 && d->head_dim <= 256, "%s: head size %lld (1..256 supported)", who, (long long)d->head_dim);
    // in the type of the sums, where it is folded with log2 e
    const double c = d->scale * LOG2E;
    NNVB_REQUIRE(std::isfinite(c) && c > 0 && (d->dtype == NNVB_F64 || (std::isfinite(float(c)) && float(c) > 0)),
                 "%s: the factor on the scores must be finite and positive", who);
    for (const int64_t* s : {d->q_stride, d->k_stride, d->v_stride, d->out_stride, d->dout_stride})
        for (int i = 0; i < 3; ++i) NNVB_REQUIRE(s[i] >= 0, "%s: negative stride", who);
    return NNVB_OK;
}

// the rows of a written tensor must lie apart
int check_out(const char* who, const nnvb_attention_desc* d) {
    const int64_t n[3] = {d->batch, d->q_len, d->q_heads};
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int x, int y) { return d->out_stride[x] < d->out_stride[y]; });
    int64_t span = d->head_dim;            // elements from the first to behind the last, over the dimensions so far
    for (int i : order) {
        if (n[i] <= 1) continue;
        NNVB_REQUIRE(d->out_stride[i] >= span, "%s: the rows of the output overlap", who);
        span += d->out_stride[i] * (n[i] - 1);
    }
    return NNVB_OK;
}

AttnArgs make_args(const nnvb_attention_desc* d) {
    AttnArgs a{};
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = d->q_stride[i]; a.ks[i] = d->k_stride[i]; a.vs[i] = d->v_stride[i];
        a.os[i] = d->out_stride[i]; a.dos[i] = d->dout_stride[i];
    }
    // the stride of a dimension of one entry says nothing
    const int64_t nq[3] = {d->batch, d->q_len, d->q_heads}, nk[3] = {d->batch, d->kv_len, d->kv_heads};
    for (int i = 0; i < 3; ++i) {
        if (nq[i] == 1) a.qs[i] = a.os[i] = a.dos[i] = 0;
        if (nk[i] == 1) a.ks[i] = a.vs[i] = 0;
    }
    a.B = int(d->batch); a.Lq = int(d->q_len); a.Lk = int(d->kv_len);
    a.Hq = int(d->q_heads); a.Hkv = int(d->kv_heads); a.D = int(d->head_dim);
    a.scale = d->scale;
    a.dtype = d->dtype;
    return a;
}

}  // namespace

extern "C" {

int nnvb_cross_attention_forward(void* stream, const nnvb_attention_desc* d, const void* q, const void* k, const void* v,
                                 const int32_t* lengths, void* out, void* lse) {
    NNVB_TRY(check_desc("nnvb_cross_attention_forward", d));
    NNVB_TRY(check_out("nnvb_cross_attention_forward", d));
    if (d->batch == 0 || d->q_len == 0) return NNVB_OK;
    NNVB_REQUIRE(q && out && (d->kv_len == 0 || (k && v)), "nnvb_cross_attention_forward: NULL pointer");
    AttnArgs a = make_args(d);
    a.q = q; a.k = k; a.v = v; a.o = out; a.lse = lse; a.lengths = lengths;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (attn_rows_takes(a)) return attn_forward_rows(st, a);
    if ((d->dtype == NNVB_F64 || d->dtype == NNVB_F32) && d->head_dim <= 128) return attn_forward_wide(st, a);
    return attn_tc_takes_forward(a) ? attn_forward_tc(st, a) : attn_forward_simt(st, a);
}

int64_t nnvb_cross_attention_workspace(const nnvb_attention_desc* d) {
    if (!d || d->batch < 0 || d->q_len < 0 || d->q_heads < 0) return 0;
    // delta, and for the tensor cores the log-sum-exp beside it, in rows padded to a tile
    const int64_t rows = d->batch * d->q_heads * round_up(d->q_len, 64), stats = rows * 8;
    if (d->dtype != NNVB_F16 || d->kv_heads < 0 || d->kv_len < 0) return stats;
    // the norms that bound dS: of dO's rows, one of 16, and of V's states
    return stats + round_up((rows / 16 + d->batch * d->kv_heads * ceil_div(d->kv_len, V_CHUNK)) * 4, 16);
}

int nnvb_cross_attention_backward(void* stream, const nnvb_attention_desc* d, const void* dout, const void* q,
                                  const void* k, const void* v, const void* out, const void* lse,
                                  const int32_t* lengths, void* dq, void* dk, void* dv, void* workspace,
                                  int64_t workspace_bytes) {
    NNVB_TRY(check_desc("nnvb_cross_attention_backward", d));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d->batch == 0) return NNVB_OK;
    const size_t e = size_t(dtype_bytes(d->dtype));
    const size_t nq = size_t(d->batch * d->q_len * d->q_heads * d->head_dim) * e;
    const size_t nk = size_t(d->batch * d->kv_len * d->kv_heads * d->head_dim) * e;
    NNVB_REQUIRE((nq == 0 || dq) && (nk == 0 || (dk && dv)), "nnvb_cross_attention_backward: NULL pointer");
    if (nq == 0 || nk == 0) {              // one side is empty: nothing reaches the other
        if (nq) NNVB_CUDA(cudaMemsetAsync(dq, 0, nq, st));
        if (nk) {
            NNVB_CUDA(cudaMemsetAsync(dk, 0, nk, st));
            NNVB_CUDA(cudaMemsetAsync(dv, 0, nk, st));
        }
        return NNVB_OK;
    }
    NNVB_REQUIRE(dout && q && k && v && out && lse, "nnvb_cross_attention_backward: NULL pointer");
    NNVB_REQUIRE(workspace && workspace_bytes >= nnvb_cross_attention_workspace(d) &&
                     reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                 "nnvb_cross_attention_backward: needs a 16-byte aligned workspace of %lld bytes",
                 (long long)nnvb_cross_attention_workspace(d));
    AttnArgs a = make_args(d);
    a.dout = dout; a.q = q; a.k = k; a.v = v; a.o = out; a.lse = const_cast<void*>(lse); a.lengths = lengths;
    a.dq = dq; a.dk = dk; a.dv = dv; a.delta = workspace;
    if (attn_tc_takes_backward(a)) return attn_backward_tc(st, a);
    NNVB_TRY(attn_delta(st, a));
    // Large problems have the wide kernels' throughput (8 x 512 x 1024 x 8 x 64 double: 1.5 against 2.5 ms; 8 x 1024 x 2048 x 16 x
    // 64 float: 6.3 against 7.4 ms).  Where one side is short, or tiles are fewer than the SMs need, the blocks of twice as many
    // threads on smaller tiles are the faster ones (2 x 3582 x 8 x 8 x 4 x 64 double: 0.79 against 0.94 ms).  More than 64
    // float channels leave a wide block alone on its SM: there both of its kernels need the tiles (4 x 148 x 677 x 12 x 96
    // float, 144 and 528 tiles: 342 wide, 377 us not; 2 x 127 x 198 x 16 x 2 x 80 double: 352 and 435).
    const int64_t heads = int64_t(a.B) * a.Hkv, rows = int64_t(a.Lq) * (a.Hq / a.Hkv);
    const int64_t tq = ceil_div(rows, 64) * heads, tk = ceil_div(a.Lk, 64) * heads;
    const bool wide = (a.dtype == NNVB_F64 || a.dtype == NNVB_F32) && a.D <= 128 && std::min<int64_t>(rows, a.Lk) > 32 &&
                      (a.D <= 64 || a.dtype == NNVB_F64 ? std::max(tq, tk) : std::min(tq, tk)) >= 100;
    return wide ? attn_backward_wide(st, a) : attn_backward_simt(st, a);
}

}  // extern "C"
