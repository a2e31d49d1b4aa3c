// The loss head (oxz_head_*): softmax cross entropy over a large vocabulary with its gradients, without keeping the logits.
//
//   l = X W^T      loss_i = log sum_v exp(l_iv - m_i) - (l_it - m_i)      G_iv = w_i (exp(l_iv - m_i) / s_i - [v = t_i])
//   dX = c G W     dW = c G^T X
//
// One pass over the vocabulary gives each row's largest logit m_i and s_i = sum_v exp(l_iv - m_i). The gradients take the
// vocabulary in pieces: a piece's logits are formed again, turned into G on the way out of the product, and G's two products
// follow while the piece is in the workspace. Rows that are not scored take no part: the scored ones are listed first, and
// every product runs over the list.
#include <algorithm>
#include <cmath>

#include "oxz_elem.cuh"
#include "oxz_internal.h"

namespace oxz {

// What k_head_rows finds out about a batch.
struct HeadMeta {
    uint32_t n;          // scored rows
    uint32_t done;       // blocks of k_head_finish that have added their part (put back to 0 by the last)
    double weight_sum;   // of the scored rows
};

}  // namespace oxz

struct oxz_head {
    oxz_head_desc d{};
    bool allocated = false;
    uint64_t bytes = 0;
    uint64_t piece = 0;              // columns of the vocabulary in a piece
    int32_t* row_of = nullptr;       // [max_rows] slot -> row of the batch, scored rows in order
    int32_t* slot_of = nullptr;      // [max_rows] row -> slot, -1: not scored
    float2* part = nullptr;          // [tiles][max_rows] {max, sum of exp} of a slot over one tile of the vocabulary
    float* target_logit = nullptr;   // [max_rows] by slot
    float2* stats = nullptr;         // [max_rows] by row, where the caller keeps none
    double* loss_part = nullptr;     // [blocks of k_head_finish]
    oxz::HeadMeta* meta = nullptr;
    float* g = nullptr;              // [max_rows][piece]
    float* dx = nullptr;             // [max_rows][hidden] sum over the pieces
    oxz::StreamOrder order;
};

namespace oxz {
namespace {

constexpr int FINISH_ROWS = 8;  // rows a block of k_head_finish takes: one per warp

// ---- the scored rows, in order. One block: each thread counts a run of rows, a scan over the threads places them.
__global__ void __launch_bounds__(1024) k_head_rows(const int64_t* __restrict__ targets, const float* __restrict__ mask, uint32_t rows,
                                                    uint64_t vocab, int32_t* row_of, int32_t* slot_of, HeadMeta* meta) {
    __shared__ uint32_t scan[32];
    __shared__ double wsum[32];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const uint32_t each = (rows + 1023) / 1024;
    const uint32_t lo = min(rows, threadIdx.x * each), hi = min(rows, lo + each);
    uint32_t count = 0;
    double w = 0.0;
    auto scored = [&](uint32_t i) { return (mask == nullptr || mask[i] != 0.f) && (uint64_t)targets[i] < vocab; };
    for (uint32_t i = lo; i < hi; i++)
        if (scored(i)) {
            count++;
            w += mask ? (double)mask[i] : 1.0;
        }
    uint32_t inc = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= (uint32_t)o) inc += up;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if (lane == 31) scan[warp] = inc;
    if (lane == 0) wsum[warp] = w;
    __syncthreads();
    if (warp == 0) {
        uint32_t v = scan[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= (uint32_t)o) v += up;
        }
        scan[lane] = v;
        if (lane == 31) {
            double total = 0.0;
            for (int k = 0; k < 32; k++) total += wsum[k];
            meta->n = v;
            meta->done = 0;
            meta->weight_sum = total;
        }
    }
    __syncthreads();
    uint32_t at = inc - count + (warp ? scan[warp - 1] : 0);
    for (uint32_t i = lo; i < hi; i++) {
        const bool yes = scored(i);
        slot_of[i] = yes ? (int32_t)at : -1;
        if (yes) row_of[at++] = (int32_t)i;
    }
}

// {max, sum of exp(x - max)} of two sets together. An empty set is {-inf, 0}.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    if (m == -INFINITY) return make_float2(m, a.y + b.y);
    return make_float2(m, a.y * expf(a.x - m) + b.y * expf(b.x - m));
}

// ---- a row's statistics from its tiles', its loss, and the totals (by the block that ends last, in block order)
__global__ void __launch_bounds__(32 * FINISH_ROWS) k_head_finish(uint32_t rows, uint32_t pitch, uint32_t tiles, const int32_t* __restrict__ slot_of,
                                                                  const float2* __restrict__ part, const float* __restrict__ target_logit,
                                                                  const float* __restrict__ mask, float2* stats, float* row_loss,
                                                                  double* loss_part, HeadMeta* meta, float* totals) {
    __shared__ double mine[FINISH_ROWS];
    __shared__ uint32_t last;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, row = blockIdx.x * FINISH_ROWS + warp;
    if (row < rows) {
        const int32_t slot = slot_of[row];
        float2 s = make_float2(-INFINITY, 0.f);
        if (slot >= 0)
            for (uint32_t t = lane; t < tiles; t += 32) s = join(s, part[(uint64_t)t * pitch + slot]);
#pragma unroll
        for (int o = 16; o; o >>= 1) s = join(s, make_float2(__shfl_xor_sync(0xffffffffu, s.x, o), __shfl_xor_sync(0xffffffffu, s.y, o)));
        if (lane == 0) {
            const float loss = slot >= 0 ? logf(s.y) - (target_logit[slot] - s.x) : 0.f;
            stats[row] = slot >= 0 ? s : make_float2(0.f, 0.f);
            if (row_loss) row_loss[row] = loss;
            mine[warp] = slot >= 0 ? (mask ? (double)mask[row] : 1.0) * (double)loss : 0.0;
        }
    } else if (lane == 0) {
        mine[warp] = 0.0;
    }
    if (!totals) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        for (int w = 0; w < FINISH_ROWS; w++) sum += mine[w];
        loss_part[blockIdx.x] = sum;
        __threadfence();
        last = atomicAdd(&meta->done, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last || warp) return;
    __threadfence();
    double sum = 0.0;
    for (uint32_t b = lane; b < gridDim.x; b += 32) sum += __ldcg(&loss_part[b]);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
        totals[0] = (float)sum;
        totals[1] = (float)meta->weight_sum;
        meta->done = 0;
    }
}

// ---- the four products, one output tile of 64 x 64 per block, summed in f32 over steps of 16
enum Product { LOGITS_STATS, LOGITS_GRAD, D_HIDDEN, D_WEIGHT };
struct ProductArgs {
    const HeadMeta* meta;
    const int32_t* row_of;
    const void* x;
    uint64_t x_stride;
    const void* w;
    uint32_t hidden, vocab, first, columns, pitch, tiles;  // the piece [first, first + columns) of the vocabulary
    const int64_t* targets;
    const float* mask;
    const float2* stats;
    float2* part;
    float* target_logit;
    float* g;
    float* dx;
    void* dw;
    float scale;
    int accumulate, add;
};

template <typename T, typename G, int P>
__global__ void __launch_bounds__(256) k_head_product(const ProductArgs a) {
    __shared__ float sa[16][65], sb[16][65];
    const uint32_t n = a.meta->n, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const uint32_t i0 = blockIdx.y * 64, j0 = blockIdx.x * 64;
    const uint32_t M = P == D_WEIGHT ? a.columns : n, N = P == LOGITS_STATS || P == LOGITS_GRAD ? a.columns : a.hidden;
    const uint32_t K = P == D_HIDDEN ? a.columns : P == D_WEIGHT ? n : a.hidden;
    if (i0 >= M) return;
    const T* x = static_cast<const T*>(a.x);
    const T* w = static_cast<const T*>(a.w);
    float acc[4][4] = {};
    for (uint32_t k0 = 0; k0 < K; k0 += 16) {
        for (uint32_t e = threadIdx.x; e < 1024; e += 256) {
            // the faster index runs along memory
            const bool k_fast = P == LOGITS_STATS || P == LOGITS_GRAD || P == D_HIDDEN;
            const uint32_t k = k_fast ? e & 15 : e >> 6, i = k_fast ? e >> 4 : e & 63;
            float v = 0.f;
            if (k0 + k < K && i0 + i < M) {
                if (P == D_HIDDEN) v = a.g[(uint64_t)(i0 + i) * a.columns + k0 + k];
                else if (P == D_WEIGHT) v = a.g[(uint64_t)(k0 + k) * a.columns + i0 + i];
                else v = to_f32<T>(x[(uint64_t)a.row_of[i0 + i] * a.x_stride + k0 + k]);
            }
            sa[k][i] = v;
            const bool bk_fast = P == LOGITS_STATS || P == LOGITS_GRAD;
            const uint32_t kb = bk_fast ? e & 15 : e >> 6, j = bk_fast ? e >> 4 : e & 63;
            v = 0.f;
            if (k0 + kb < K && j0 + j < N) {
                if (P == D_HIDDEN) v = to_f32<T>(w[(uint64_t)(a.first + k0 + kb) * a.hidden + j0 + j]);
                else if (P == D_WEIGHT) v = to_f32<T>(x[(uint64_t)a.row_of[k0 + kb] * a.x_stride + j0 + j]);
                else v = to_f32<T>(w[(uint64_t)(a.first + j0 + j) * a.hidden + k0 + kb]);
            }
            sb[kb][j] = v;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; k++) {
            float p[4], q[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                p[r] = sa[k][ty * 4 + r];
                q[r] = sb[k][tx * 4 + r];
            }
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int c = 0; c < 4; c++) acc[r][c] = fmaf(p[r], q[c], acc[r][c]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const uint32_t i = i0 + ty * 4 + r;
        const bool in = i < M;
        const uint32_t row = in && P != D_WEIGHT ? (uint32_t)a.row_of[i] : 0;
        if (P == LOGITS_STATS) {
            const int64_t t = in ? a.targets[row] : -1;
            float2 s = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint32_t v = j0 + tx * 4 + c;
                if (in && v < N) {
                    s.x = fmaxf(s.x, acc[r][c]);
                    if ((int64_t)v == t) a.target_logit[i] = acc[r][c];
                }
            }
#pragma unroll
            for (int o = 8; o; o >>= 1) s.x = fmaxf(s.x, __shfl_xor_sync(0xffffffffu, s.x, o));
            const float ref = s.x == -INFINITY ? 0.f : s.x;
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (j0 + tx * 4 + c < N) s.y += expf(acc[r][c] - ref);
#pragma unroll
            for (int o = 8; o; o >>= 1) s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
            if (in && tx == 0) a.part[(uint64_t)blockIdx.x * a.pitch + i] = s;
        } else if (in) {
            const float2 s = P == LOGITS_GRAD ? a.stats[row] : make_float2(0.f, 0.f);
            const float weight = P == LOGITS_GRAD && a.mask ? a.mask[row] : 1.f;
            const int64_t t = P == LOGITS_GRAD ? a.targets[row] : -1;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint32_t j = j0 + tx * 4 + c;
                if (j >= N) continue;
                if (P == LOGITS_GRAD) {
                    const float e = expf(acc[r][c] - s.x);
                    a.g[(uint64_t)i * a.columns + j] = weight * ((int64_t)(a.first + j) == t ? (e - s.y) / s.y : e / s.y);
                } else if (P == D_HIDDEN) {
                    float* to = a.dx + (uint64_t)i * a.hidden + j;
                    *to = a.add ? *to + acc[r][c] : acc[r][c];
                } else {
                    G* to = static_cast<G*>(a.dw) + (uint64_t)(a.first + i) * a.hidden + j;
                    *to = from_f32<G>(a.accumulate ? to_f32<G>(*to) + acc[r][c] * a.scale : acc[r][c] * a.scale);
                }
            }
        }
    }
}

// ---- d_hidden: the scored rows' sums times the scale, rounded; zeros for the others
template <typename T>
__global__ void __launch_bounds__(256) k_head_d_hidden(uint32_t rows, uint32_t hidden, const int32_t* __restrict__ slot_of,
                                                       const float* __restrict__ dx, float scale, T* out, uint64_t stride) {
    const uint64_t total = (uint64_t)rows * hidden;
    for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (uint64_t)gridDim.x * 256) {
        const uint32_t row = (uint32_t)(e / hidden), col = (uint32_t)(e - (uint64_t)row * hidden);
        const int32_t slot = slot_of[row];
        out[(uint64_t)row * stride + col] = from_f32<T>(slot < 0 ? 0.f : dx[(uint64_t)slot * hidden + col] * scale);
    }
}

bool misaligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) % to) != 0; }

template <typename T, typename G, int P>
void product(const ProductArgs& a, uint64_t m, uint64_t n, cudaStream_t s) {
    if (m && n) k_head_product<T, G, P><<<dim3((unsigned)((n + 63) / 64), (unsigned)((m + 63) / 64)), 256, 0, s>>>(a);
}

template <typename T, typename G>
int32_t run(oxz_head* h, const oxz_head_batch& b, float* row_loss, float2* row_stats, bool want_loss, float* totals, const oxz_head_grads* gr,
            cudaStream_t s) {
    const oxz_head_desc& d = h->d;
    k_head_rows<<<1, 1024, 0, s>>>(b.targets, b.loss_mask, (uint32_t)b.rows, d.vocab, h->row_of, h->slot_of, h->meta);
    ProductArgs a{};
    a.meta = h->meta;
    a.row_of = h->row_of;
    a.x = b.hidden;
    a.x_stride = b.hidden_stride;
    a.w = b.weight;
    a.hidden = (uint32_t)d.hidden;
    a.vocab = (uint32_t)d.vocab;
    a.pitch = (uint32_t)d.max_rows;
    a.targets = b.targets;
    a.mask = b.loss_mask;
    a.part = h->part;
    a.target_logit = h->target_logit;
    a.g = h->g;
    a.dx = h->dx;
    float2* stats = row_stats ? row_stats : h->stats;
    if (want_loss) {
        a.columns = (uint32_t)d.vocab;
        product<T, G, LOGITS_STATS>(a, b.rows, d.vocab, s);
        const unsigned blocks = std::max<unsigned>(1, (unsigned)((b.rows + FINISH_ROWS - 1) / FINISH_ROWS));
        k_head_finish<<<blocks, 32 * FINISH_ROWS, 0, s>>>((uint32_t)b.rows, a.pitch, (uint32_t)((d.vocab + 63) / 64), h->slot_of, h->part,
                                                          h->target_logit, b.loss_mask, stats, row_loss, h->loss_part, h->meta, totals);
    }
    if (gr) {
        a.stats = stats;
        a.scale = (float)gr->grad_scale;
        a.accumulate = gr->accumulate;
        a.dw = gr->d_weight;
        for (uint64_t v = 0; v < d.vocab; v += h->piece) {
            a.first = (uint32_t)v;
            a.columns = (uint32_t)std::min(h->piece, d.vocab - v);
            a.add = v > 0;
            product<T, G, LOGITS_GRAD>(a, b.rows, a.columns, s);
            if (gr->d_hidden) product<T, G, D_HIDDEN>(a, b.rows, d.hidden, s);
            if (gr->d_weight) product<T, G, D_WEIGHT>(a, a.columns, d.hidden, s);
        }
        if (gr->d_hidden && b.rows)
            k_head_d_hidden<T><<<(unsigned)std::min<uint64_t>((b.rows * d.hidden + 255) / 256, 148 * 8), 256, 0, s>>>(
                (uint32_t)b.rows, (uint32_t)d.hidden, h->slot_of, h->dx, (float)gr->grad_scale, static_cast<T*>(gr->d_hidden), gr->d_hidden_stride);
    }
    return OXZ_OK;
}

int32_t call(const char* who, oxz_head* h, const oxz_head_batch* batch, float* row_loss, float* row_stats, float* totals, bool want_loss,
             const oxz_head_grads* grads, bool want_grads, void* stream) {
    if (!h || !batch || (want_grads && !grads)) return fail(OXZ_ERR_INVALID, "%s: null argument", who);
    const oxz_head_desc& d = h->d;
    oxz_head_batch b = *batch;
    oxz_head_grads g{};
    if (want_grads) g = *grads;
    if (b.rows > d.max_rows)
        return fail(OXZ_ERR_INVALID, "%s: %llu rows, the handle was made for %llu", who, (unsigned long long)b.rows, (unsigned long long)d.max_rows);
    if (!b.weight || (b.rows && (!b.hidden || !b.targets))) return fail(OXZ_ERR_INVALID, "%s: null argument", who);
    if (!want_loss && b.rows && !row_stats) return fail(OXZ_ERR_INVALID, "%s: the gradients need the rows' statistics", who);
    if (want_grads && !g.d_hidden && !g.d_weight) return fail(OXZ_ERR_INVALID, "%s: neither d_hidden nor d_weight is wanted", who);
    if (b.hidden_stride == 0) b.hidden_stride = d.hidden;
    if (g.d_hidden_stride == 0) g.d_hidden_stride = d.hidden;
    if (b.hidden_stride < d.hidden || b.hidden_stride > (1ull << 31) || g.d_hidden_stride < d.hidden || g.d_hidden_stride > (1ull << 31))
        return fail(OXZ_ERR_INVALID, "%s: strides %llu and %llu with rows of %llu", who, (unsigned long long)b.hidden_stride,
                    (unsigned long long)g.d_hidden_stride, (unsigned long long)d.hidden);
    const size_t es = dtype_size(d.dtype);
    if (misaligned(b.hidden, es) || misaligned(b.targets, 8) || misaligned(b.loss_mask, 4) || misaligned(g.d_hidden, es) || misaligned(row_loss, 4) ||
        misaligned(row_stats, 8) || misaligned(totals, 4))
        return fail(OXZ_ERR_INVALID, "%s: a pointer is not aligned to its element", who);
    if (misaligned(b.weight, 16) || misaligned(g.d_weight, 16)) return fail(OXZ_ERR_INVALID, "%s: weight and d_weight are aligned to 16 bytes", who);
    if (want_grads && !std::isfinite((float)g.grad_scale)) return fail(OXZ_ERR_INVALID, "%s: grad_scale %g is not a finite f32", who, g.grad_scale);
    if (!h->allocated) return fail(OXZ_ERR_STATE, "%s: no workspace: call oxz_head_alloc first", who);
    DeviceGuard dev;
    OXZ_TRY(dev.enter(d.device));
    cudaStream_t s = (cudaStream_t)stream;
    OXZ_TRY(h->order.begin(s));
    float2* st = reinterpret_cast<float2*>(row_stats);
    const oxz_head_grads* gp = want_grads ? &g : nullptr;
    int32_t rc;
    if (d.dtype == OXZ_F32) rc = run<float, float>(h, b, row_loss, st, want_loss, totals, gp, s);
    else if (d.dtype == OXZ_BF16 && d.grad_dtype == OXZ_F32) rc = run<__nv_bfloat16, float>(h, b, row_loss, st, want_loss, totals, gp, s);
    else if (d.dtype == OXZ_BF16) rc = run<__nv_bfloat16, __nv_bfloat16>(h, b, row_loss, st, want_loss, totals, gp, s);
    else if (d.grad_dtype == OXZ_F32) rc = run<__half, float>(h, b, row_loss, st, want_loss, totals, gp, s);
    else rc = run<__half, __half>(h, b, row_loss, st, want_loss, totals, gp, s);
    OXZ_TRY(rc);
    OXZ_CUDA(cudaGetLastError());
    return h->order.end(s);
}

}  // namespace
}  // namespace oxz

using namespace oxz;

extern "C" {

int32_t oxz_head_create(const oxz_head_desc* desc, oxz_head** out) {
    return guarded("oxz_head_create", [&]() -> int32_t {
        if (!desc || !out) return fail(OXZ_ERR_INVALID, "oxz_head_create: null argument");
        *out = nullptr;
        const oxz_head_desc& d = *desc;
        if (d.max_rows == 0 || d.max_rows > 0x7fffffffull)
            return fail(OXZ_ERR_INVALID, "oxz_head_create: max_rows %llu is outside 1..2^31-1", (unsigned long long)d.max_rows);
        if (d.vocab == 0 || d.vocab > 0x7fffffffull)
            return fail(OXZ_ERR_INVALID, "oxz_head_create: vocab %llu is outside 1..2^31-1", (unsigned long long)d.vocab);
        if (d.hidden == 0 || d.hidden > (1u << 20))
            return fail(OXZ_ERR_INVALID, "oxz_head_create: hidden %llu is outside 1..2^20", (unsigned long long)d.hidden);
        if (d.dtype != OXZ_F32 && d.dtype != OXZ_BF16 && d.dtype != OXZ_F16)
            return fail(OXZ_ERR_INVALID, "oxz_head_create: dtype %d is none of f32, bf16, f16", d.dtype);
        if (d.grad_dtype != d.dtype && d.grad_dtype != OXZ_F32)
            return fail(OXZ_ERR_INVALID, "oxz_head_create: grad_dtype %d is neither the dtype (%d) nor f32", d.grad_dtype, d.dtype);
        if (d.device < 0) return fail(OXZ_ERR_INVALID, "oxz_head_create: device %d", d.device);
        oxz_head* h = new oxz_head();
        h->d = d;
        *out = h;
        return OXZ_OK;
    });
}

int32_t oxz_head_alloc(oxz_head* h, uint64_t* workspace_bytes) {
    return guarded("oxz_head_alloc", [&]() -> int32_t {
        if (!h) return fail(OXZ_ERR_INVALID, "oxz_head_alloc: null handle");
        if (!h->allocated) {
            DeviceGuard dev;
            OXZ_TRY(dev.enter(h->d.device));
            const oxz_head_desc& d = h->d;
            const uint64_t limit = d.piece_bytes ? d.piece_bytes : 512ull << 20;
            h->piece = std::min<uint64_t>(d.vocab, std::max<uint64_t>(64, limit / (d.max_rows * 4) / 64 * 64));
            uint64_t bytes = 0;
            auto get = [&](auto** p, uint64_t n) -> int32_t {  // what a failed attempt left behind is kept and used by the next one
                if (!*p) OXZ_CUDA(cudaMalloc((void**)p, n));
                bytes += n;
                return OXZ_OK;
            };
            OXZ_TRY(get(&h->row_of, d.max_rows * 4));
            OXZ_TRY(get(&h->slot_of, d.max_rows * 4));
            OXZ_TRY(get(&h->part, (d.vocab + 63) / 64 * d.max_rows * 8));
            OXZ_TRY(get(&h->target_logit, d.max_rows * 4));
            OXZ_TRY(get(&h->stats, d.max_rows * 8));
            OXZ_TRY(get(&h->loss_part, (d.max_rows + FINISH_ROWS - 1) / FINISH_ROWS * 8));
            OXZ_TRY(get(&h->meta, sizeof(HeadMeta)));
            OXZ_TRY(get(&h->g, d.max_rows * h->piece * 4));
            OXZ_TRY(get(&h->dx, d.max_rows * d.hidden * 4));
            OXZ_TRY(h->order.create());
            h->bytes = bytes;
            h->allocated = true;
        }
        if (workspace_bytes) *workspace_bytes = h->bytes;
        return OXZ_OK;
    });
}

int32_t oxz_head_destroy(oxz_head* h) {
    return guarded("oxz_head_destroy", [&]() -> int32_t {
        if (!h) return OXZ_OK;
        DeviceGuard dev;
        if (h->row_of) dev.enter(h->d.device);
        h->order.destroy();
        for (void* p : {(void*)h->row_of, (void*)h->slot_of, (void*)h->part, (void*)h->target_logit, (void*)h->stats, (void*)h->loss_part,
                        (void*)h->meta, (void*)h->g, (void*)h->dx})
            if (p) cudaFree(p);
        delete h;
        return OXZ_OK;
    });
}

int32_t oxz_head_loss_async(oxz_head* h, const oxz_head_batch* batch, float* row_loss, float* row_stats, float* totals, void* stream) {
    return guarded("oxz_head_loss_async", [&]() -> int32_t { return call("oxz_head_loss_async", h, batch, row_loss, row_stats, totals, true, nullptr, false, stream); });
}

int32_t oxz_head_grads_async(oxz_head* h, const oxz_head_batch* batch, const float* row_stats, const oxz_head_grads* grads, void* stream) {
    return guarded("oxz_head_grads_async", [&]() -> int32_t {
        return call("oxz_head_grads_async", h, batch, nullptr, const_cast<float*>(row_stats), nullptr, false, grads, true, stream);
    });
}

int32_t oxz_head_loss_grads_async(oxz_head* h, const oxz_head_batch* batch, float* row_loss, float* row_stats, float* totals,
                                  const oxz_head_grads* grads, void* stream) {
    return guarded("oxz_head_loss_grads_async", [&]() -> int32_t {
        return call("oxz_head_loss_grads_async", h, batch, row_loss, row_stats, totals, true, grads, true, stream);
    });
}

}  // extern "C"
