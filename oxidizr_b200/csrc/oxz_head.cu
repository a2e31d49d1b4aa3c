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
#include <atomic>
#include <cmath>
#include <type_traits>

#include <cuda.h>

#include "oxz_elem.cuh"
#include "oxz_head_few.cuh"
#include "oxz_internal.h"
#include "oxz_tcgen05.cuh"

namespace oxz {

// What k_head_rows finds out about a batch.
struct HeadMeta {
    uint32_t n;          // scored rows
    uint32_t done;       // blocks of k_head_finish that have added their part (put back to 0 by the last)
    double weight_sum;   // of the scored rows
    float up, down;      // power of two G is scaled by before it is rounded (f16 only), and its inverse
    uint32_t kept;       // columns of a row of `l` where the losses leave the logits for the gradients; 0: they do not all fit
};

}  // namespace oxz

struct oxz_head {
    oxz_head_desc d{};
    bool allocated = false;
    uint64_t bytes = 0;
    uint64_t piece = 0;              // columns of the vocabulary in a piece
    int32_t* row_of = nullptr;       // [max_rows] slot -> row of the batch, scored rows in order
    int32_t* slot_of = nullptr;      // [max_rows] row -> slot, -1: not scored
    float2* part = nullptr;          // [2 * tiles][rows] {max, sum of exp} of a slot over half a tile of the vocabulary
    float* target_logit = nullptr;   // [max_rows] by slot
    float2* stats = nullptr;         // [max_rows] by row, where the caller keeps none
    double* loss_part = nullptr;     // [blocks of k_head_finish]
    oxz::HeadMeta* meta = nullptr;
    uint64_t cap = 0;                // max_rows up to a multiple of a tile
    uint32_t pitch = 0;              // elements of a packed row: hidden up to 16 bytes
    uint32_t dx_pitch = 0;           // of a row of dx
    int parts = 1, g_parts = 1;      // 16-bit parts of an operand, and of G
    int clusters = 0;                // pairs of SMs the device runs at once
    void* x = nullptr;               // [parts][cap][pitch] packed hidden states
    void* w = nullptr;               // [parts][vocab][pitch] packed weight, where TMA cannot read the caller's
    void* g = nullptr;               // [g_parts][piece / 64][cap][64]: every box that is written or read is one stretch of memory
    float* l = nullptr;              // [scored rows][kept] logits
    uint64_t l_elems = 0, kept_pitch = 0;
    bool keep_large = false;         // also batches of more than FEW_LOGITS logits keep them
    float* dx = nullptr;             // [scored rows][dx_pitch] sums over the pieces
    float* dx_shares = nullptr;      // tiles of 256 x 256: the shares after the first of the tiles that are cut
    int sms = 0;
    float* few_logits = nullptr;     // [vocab][R]: the path for a handful of rows
    float2* few_part = nullptr;
    float* few_dx = nullptr;
    uint32_t* few_done = nullptr;
    int32_t* expired = nullptr;      // mapped host memory: a bounded wait inside a kernel ran out
    int32_t* d_expired = nullptr;
    oxz::StreamOrder order;
};

namespace oxz {
namespace {

constexpr uint64_t FEW_LOGITS = 1ull << 22;
constexpr uint32_t FINISH_ROWS = 8;  // rows a block of k_head_finish takes at least
constexpr uint32_t MMA_M = 256, MMA_N = 256, MMA_K = 64;  // tile of a pair of SMs (the logits' may be narrower: see tile_width)

__host__ __device__ inline uint32_t tiles_of(uint64_t n, uint32_t of) { return (uint32_t)((n + of - 1) / of); }

__device__ __forceinline__ void describe(HeadMeta* meta, uint32_t n, double weight_sum, float top, int f16, uint64_t vocab, uint64_t l_elems) {
    meta->n = n;
    meta->done = 0;
    meta->weight_sum = weight_sum;
    // f16 holds 2^-24 .. 65504: the largest weight times one goes to 2^13 .. 2^14, so that probabilities down to 2^-27 of it stay
    // normal numbers
    const int up = f16 && top > 0.f && isfinite(top) ? min(max(13 - ilogbf(top), -100), 100) : 0;
    meta->up = exp2f((float)up);
    meta->down = exp2f((float)-up);
    const uint64_t all = (vocab + MMA_N - 1) / MMA_N * MMA_N;
    meta->kept = n * all <= l_elems ? (uint32_t)all : 0;
}

// ---- the scored rows, in order, and what the other kernels need to know of them. One block: a warp takes a contiguous run of rows,
// 32 at a time; a scan over the warps' counts places them.
__global__ void __launch_bounds__(1024) k_head_rows(const int64_t* __restrict__ targets, const float* __restrict__ mask, uint32_t rows,
                                                    uint64_t vocab, int32_t* row_of, int32_t* slot_of, HeadMeta* meta, int f16,
                                                    uint64_t l_elems) {
    let_next();
    __shared__ uint32_t counts[32];
    __shared__ double wsum[32];
    __shared__ float wtop[32];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const uint32_t turns = (rows + 1023) / 1024;
    const uint64_t begin = (uint64_t)warp * turns * 32;
    auto weight = [&](uint64_t i) { return i < rows && (uint64_t)targets[i] < vocab ? (mask ? mask[i] : 1.f) : 0.f; };
    uint32_t count = 0, kept_bits = 0;  // lane k keeps the flags of turn k: the second walk of up to 32 turns reads nothing again
    double sum = 0.0;
    float top = 0.f;
    for (uint32_t t = 0; t < turns; t++) {
        const float w = weight(begin + (uint64_t)t * 32 + lane);
        const uint32_t bits = __ballot_sync(0xffffffffu, w != 0.f);
        if (t == lane) kept_bits = bits;
        count += __popc(bits);
        sum += (double)w;
        top = fmaxf(top, fabsf(w));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (lane == 0) {
        counts[warp] = count;
        wsum[warp] = sum;
        wtop[warp] = top;
    }
    __syncthreads();
    uint32_t at = 0, n = 0;
    for (uint32_t w = 0; w < 32; w++) {
        at += w < warp ? counts[w] : 0;
        n += counts[w];
    }
    if (threadIdx.x == 0) {
        double total = 0.0;
        for (int k = 0; k < 32; k++) {
            total += wsum[k];
            top = fmaxf(top, wtop[k]);
        }
        describe(meta, n, total, top, f16, vocab, l_elems);
    }
    for (uint32_t t = 0; t < turns; t++) {
        const uint64_t i = begin + (uint64_t)t * 32 + lane;
        const uint32_t bits = turns <= 32 ? __shfl_sync(0xffffffffu, kept_bits, t) : __ballot_sync(0xffffffffu, weight(i) != 0.f);
        const bool yes = bits >> lane & 1;
        const uint32_t slot = at + __popc(bits & ((1u << lane) - 1));
        if (i < rows) slot_of[i] = yes ? (int32_t)slot : -1;
        if (yes) row_of[slot] = (int32_t)i;
        at += __popc(bits);
    }
}

// ---- the rows' statistics from their tiles', their losses, and the totals (by the block that ends last, in block order). A block
// takes ROWS rows, a thread every few tiles of one of them, four at once; the threads of a row are joined in order. ROWS is 8, and 32
// for many rows: 32 would leave a batch of some hundred rows to a handful of blocks, each a long chain of loads.
template <int ROWS>
__global__ void __launch_bounds__(1024) k_head_finish(uint32_t rows, uint32_t pitch, uint32_t tiles, const int32_t* __restrict__ slot_of,
                                                      const float2* __restrict__ part, const float* __restrict__ target_logit,
                                                      const float* __restrict__ mask, float2* stats, float* row_loss, double* loss_part,
                                                      HeadMeta* meta, float* totals) {
    __shared__ float2 share[1024 / ROWS][ROWS + 1];
    __shared__ double mine[ROWS];
    __shared__ uint32_t last;
    let_next();
    after_previous();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, row = blockIdx.x * ROWS + lane % ROWS, first = threadIdx.x / ROWS;
    const int32_t slot = row < rows ? slot_of[row] : -1;
    // the row that the warp ends, asked for now
    const uint32_t own = blockIdx.x * ROWS + warp;
    const int32_t at = warp < ROWS && own < rows ? slot_of[own] : -1;
    const float own_logit = at >= 0 ? target_logit[at] : 0.f;
    const double own_weight = at >= 0 ? (mask ? (double)mask[own] : 1.0) : 0.0;
    float2 s = make_float2(-INFINITY, 0.f);
    if (slot >= 0) {
        const uint32_t step = blockDim.x / ROWS;
        for (uint32_t t = first; t < tiles; t += 4 * step) {
            float2 p[4];
#pragma unroll
            for (int k = 0; k < 4; k++) p[k] = t + step * k < tiles ? part[(uint64_t)(t + step * k) * pitch + slot] : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int k = 0; k < 4; k++) s = join_stats(s, p[k]);
        }
    }
    share[first][lane % ROWS] = s;
    __syncthreads();
    // now a warp has one row, a lane four of its parts
    if (warp < ROWS) {
        s = share[lane][warp];
        for (uint32_t k = lane + 32; k < blockDim.x / ROWS; k += 32) s = join_stats(s, share[k][warp]);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) s = join_stats(s, make_float2(__shfl_xor_sync(0xffffffffu, s.x, o), __shfl_xor_sync(0xffffffffu, s.y, o)));
        if (lane == 0) {
            const float loss = at >= 0 ? logf(s.y) - (own_logit - s.x) : 0.f;
            if (own < rows) {
                stats[own] = at >= 0 ? s : make_float2(0.f, 0.f);
                if (row_loss) row_loss[own] = loss;
            }
            mine[warp] = at >= 0 ? own_weight * (double)loss : 0.0;
        }
    }
    if (!totals) return;
    __syncthreads();
    if (warp) return;
    double sum = lane < ROWS ? mine[lane] : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (gridDim.x == 1) {
        if (lane == 0) {
            totals[0] = (float)sum;
            totals[1] = (float)meta->weight_sum;
        }
        return;
    }
    if (lane == 0) {
        loss_part[blockIdx.x] = sum;
        __threadfence();
        last = atomicAdd(&meta->done, 1u) == gridDim.x - 1;
    }
    __syncwarp();
    if (!last) return;
    __threadfence();
    sum = 0.0;
    for (uint32_t b = lane; b < gridDim.x; b += 32) sum += __ldcg(&loss_part[b]);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
        totals[0] = (float)sum;
        totals[1] = (float)meta->weight_sum;
        meta->done = 0;
    }
}

// ---- the scored rows' hidden states, packed for the products: [part][slot][pitch] 16-bit values, zeros to the end of the pitch and
// in the rows up to the next multiple of a tile, which the products read. An f32 is the sum of three bf16 of 8 bits each (cut, not
// rounded, so that no part leaves the range); 16-bit values are copied.
template <typename T, typename S>
__device__ __forceinline__ void pack_piece(const float (&v)[8], S* out, uint64_t part_stride, int parts) {
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; j++) rest[j] = v[j];
    for (int p = 0; p < parts; p++) {
        Vec<S, 8> o;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if constexpr (sizeof(T) == 4) {
                float hi = __uint_as_float(__float_as_uint(rest[j]) & 0xffff0000u);
                rest[j] = isfinite(v[j]) ? rest[j] - hi : 0.f;  // an infinity or a NaN is its first part alone
                // no part of a value is zero where the value is not: times an infinity it would make a NaN of it
                if (hi == 0.f && isfinite(v[j]) && fabsf(v[j]) > 0x1p-100f) hi = copysignf(0x1p-126f, v[j]);
                o.e[j] = from_f32<S>(hi);
            } else {
                o.e[j] = from_f32<S>(v[j]);
            }
        }
        o.store(out + p * part_stride);
    }
}
template <typename T, typename S>
__device__ __forceinline__ void pack_at(const T* src, bool here, uint32_t col, uint32_t hidden, int wide, S* out, uint64_t part_stride, int parts) {
    float v[8];
    if (!here) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0.f;
    } else if (wide && col + 8 <= hidden) {
        Vec<T, 8> x;
        x.load(src + col);
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = to_f32<T>(x.e[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = col + j < hidden ? to_f32<T>(src[col + j]) : 0.f;
    }
    pack_piece<T, S>(v, out, part_stride, parts);
}
// rows: the packed rows (row_of null: row i is source row i, `rows` of them; else the scored ones and zeros to the next multiple of 256)
template <typename T, typename S>
__global__ void __launch_bounds__(256) k_head_pack(const T* __restrict__ src, uint64_t stride, uint32_t hidden, uint32_t pitch, uint64_t rows,
                                                   const int32_t* __restrict__ row_of, const HeadMeta* __restrict__ meta, S* out,
                                                   uint64_t part_stride, int parts, int wide) {
    let_next();
    after_previous();
    const uint32_t n = row_of ? meta->n : (uint32_t)rows, per = pitch / 8;
    const uint64_t total = (row_of ? (uint64_t)tiles_of(n, MMA_M) * MMA_M : rows) * per;
    for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (uint64_t)gridDim.x * 256) {
        const uint64_t slot = e / per;
        const uint32_t col = (uint32_t)(e - slot * per) * 8;
        const bool here = slot < n;
        pack_at<T, S>(here ? src + (row_of ? (uint64_t)row_of[slot] : slot) * stride : nullptr, here, col, hidden, wide, out + slot * pitch + col,
                      part_stride, parts);
    }
}
// Up to LISTED rows: every block lists the scored ones for itself (a row a thread) and packs its share; the first leaves the list for
// the other kernels. One launch instead of two.
constexpr uint32_t LISTED = 1024;
template <typename T, typename S>
__global__ void __launch_bounds__(LISTED) k_head_list_pack(const int64_t* __restrict__ targets, const float* __restrict__ mask, uint32_t rows, uint64_t vocab,
                                                           int32_t* row_of, int32_t* slot_of, HeadMeta* meta, int f16, uint64_t l_elems,
                                                           const T* __restrict__ src, uint64_t stride, uint32_t hidden, uint32_t pitch, S* out,
                                                           uint64_t part_stride, int parts, int wide) {
    __shared__ uint32_t bits_of[32];
    __shared__ uint16_t list[LISTED];
    __shared__ double wsum[32];
    __shared__ float wtop[32];
    let_next();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, i = threadIdx.x;
    const float w = i < rows && (uint64_t)targets[i] < vocab ? (mask ? mask[i] : 1.f) : 0.f;
    const uint32_t bits = __ballot_sync(0xffffffffu, w != 0.f);
    double sum = (double)w;
    float top = fabsf(w);
    if (blockIdx.x == 0) {
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
    }
    if (lane == 0) {
        bits_of[warp] = bits;
        wsum[warp] = sum;
        wtop[warp] = top;
    }
    __syncthreads();
    uint32_t at = 0, n = 0;
    for (uint32_t k = 0; k < 32; k++) {
        const uint32_t c = __popc(bits_of[k]);
        at += k < warp ? c : 0;
        n += c;
    }
    const bool yes = bits >> lane & 1;
    at += __popc(bits & ((1u << lane) - 1));
    if (yes) list[at] = (uint16_t)i;
    if (blockIdx.x == 0) {
        if (i < rows) slot_of[i] = yes ? (int32_t)at : -1;
        if (yes) row_of[at] = (int32_t)i;
        if (i == 0) {
            double total = 0.0;
            for (int k = 0; k < 32; k++) {
                total += wsum[k];
                top = fmaxf(top, wtop[k]);
            }
            describe(meta, n, total, top, f16, vocab, l_elems);
        }
    }
    __syncthreads();
    const uint32_t per = pitch / 8, end = tiles_of(n, MMA_M) * MMA_M * per;
    for (uint32_t e = blockIdx.x * LISTED + i; e < end; e += gridDim.x * LISTED) {
        const uint32_t slot = e / per, col = (e - slot * per) * 8;
        const bool here = slot < n;
        pack_at<T, S>(here ? src + (uint64_t)list[slot] * stride : nullptr, here, col, hidden, wide, out + (uint64_t)slot * pitch + col, part_stride, parts);
    }
}

// ---- the four products on the tensor cores.
//
// A pair of SMs works on one output tile of 256 x 256 (cta_group::2): each holds 128 rows of A and of the accumulator and half of B's
// rows, so that a step of 64 in K costs an SM 32 KiB from L2 for 2 x 256 x 128 x 64 operations. One thread per SM keeps STAGES
// steps of both operands in flight by TMA, one thread of the pair issues the products, eight warps per SM take the finished tile
// from tensor memory while the other of its two buffers fills.
// The tensor cores cut, not round, what they add to an accumulator: over K = 2048 the logits lose 2e-6 of the loss, over the
// vocabulary of an f32 gradient 1e-5. Where that shows (RUN > 0) an accumulator holds RUN steps of K only and the runs are added in
// f32 registers, rounded; parts of a value are added the small ones first. A cut goes one way, so the batch's total keeps what its rows
// lose: 16-bit logits of hidden 2048 by runs of 4 are 2e-7 of the loss off, rows and total (bf16; f16 2.6e-7); runs of 8 leave
// 4.4e-7 (5.5e-7) in 1 to 2 % less time (8192 x 2048 x 128256 bf16 with gradients 13.69 ms, 13.84), runs of 2 1e-7 in 9 % more.
//   LOGITS_STATS  l = X W^T: each row's {max, sum of exp} over half a tile's columns goes out, and the target's logit
//   LOGITS_GRAD   the same tile, turned into G
//   D_HIDDEN      G W, summed over the pieces in f32; its tiles are few and long (K is a piece of the vocabulary): see Split
//   D_WEIGHT      G^T X
// Operands come as K runs in memory: G and X are K-major in the first three, W in the first two; the others are read with K along
// the lines of their tiles. Values of more than 16 bits come in parts; a product of such operands is the sum over `pairs` of parts.
enum Product { LOGITS_STATS, LOGITS_GRAD, D_HIDDEN, D_WEIGHT };
constexpr int STAGES = 5, MMA_THREADS = 320, EPILOGUE_WARPS = 8;
constexpr uint32_t STAGE_BYTES = 4 * BOX_BYTES, OUT_BYTES = 2 * 32 * 128;
constexpr uint32_t MMA_SMEM = STAGES * STAGE_BYTES + EPILOGUE_WARPS * OUT_BYTES + 1024 + 256;

struct ProductArgs {
    const HeadMeta* meta;
    const int32_t* row_of;
    uint32_t hidden, first, columns, piece, pitch, cap, g_blocks, dx_pitch, keep, width;  // the piece [first, first + columns) of the vocabulary
    const int64_t* targets;
    const float* mask;
    const float2* stats;
    float2* part;
    float* target_logit;
    void* g;
    float* l;
    float *dx, *dx_shares;
    void* dw;
    float scale;
    int accumulate, add, bf16, n_pairs;
    int boxes;   // d_weight leaves by TMA
    int beside;  // d_weight starts beside d_hidden, on which it does not depend
    uint8_t pair_a[6], pair_b[6];
    int32_t* expired;
};

// How D_HIDDEN's tiles are shared among the pairs of SMs: rounds of whole tiles while there are enough for every pair; the rest,
// fewer than the pairs, are cut in K into `shares` each, as many as fill one to four more rounds best. The pairs of a round walk K in
// step, so that what they read is read once from memory (tiles cut at any step balance as well and read G six times over: 835 -> 1035
// us a piece of 16384 words, 8192 rows, hidden 2048).
constexpr uint32_t MAX_ROUNDS = 4;
__host__ __device__ constexpr uint32_t min_share(size_t size) { return size == 4 ? 2 : 8; }  // steps of K in a share at least; one of f32 is six products
struct Split {
    uint32_t tiles, whole, rest, shares;
    __host__ __device__ Split(uint64_t rows, uint32_t hidden, uint64_t piece, uint32_t pairs, uint32_t least) {
        tiles = tiles_of(rows, MMA_M) * tiles_of(hidden, MMA_N);
        rest = tiles % pairs;
        whole = tiles - rest;
        shares = 1;
        const uint32_t top = tiles_of(piece, MMA_K) / least;
        uint32_t rounds = 1;
        for (uint32_t r = 1; rest && r <= MAX_ROUNDS; r++) {
            uint32_t k = r * pairs / rest;
            if (k > top) k = top;
            if (k * rounds > shares * r) {  // r / k of a tile's time instead of rounds / shares
                shares = k;
                rounds = r;
            }
        }
    }
    __host__ __device__ uint32_t items() const { return whole + rest * shares; }
};

// exp(x - m). f32 results take the library's exponential. For 16-bit operands the unit's 2^x is ample: it is off by 2^-22, and the
// rounding of its argument by 2^-24 |x - m| log2 e, relatively, where the operands themselves are rounded to 2^-9 or 2^-12. The
// difference is formed first: the largest logit's own term is 1 and the sums hold f32's digits (x log2 e - m log2 e in one fused
// product leaves the rounding of m log2 e in every term of a row: at logits of 200 a sure row's loss was up to 1e-5 off, and negative).
constexpr float LOG2E = 1.4426950408889634f;
template <bool EXACT> struct ExpFrom {
    float m;
    __device__ __forceinline__ explicit ExpFrom(float at) : m(at) {}
    __device__ __forceinline__ float operator()(float x) const {
        if constexpr (EXACT) return expf(x - m);
        float r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"((x - m) * LOG2E));
        return r;
    }
    // of two, the same bits as of each
    __device__ __forceinline__ float2 operator()(float2 x) const {
        if constexpr (EXACT) return make_float2(expf(x.x - m), expf(x.y - m));
        const float2 t = mul2(add2(x, make_float2(-m, -m)), make_float2(LOG2E, LOG2E));
        float2 r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(t.x));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(t.y));
        return r;
    }
};

// G from 32 logits of a row: weight * up / s * (exp(l - m) - [v = t] s). `target`, `valid`: column of the target, columns that exist,
// both counted from the first of the 32.
template <bool EXACT>
__device__ __forceinline__ void logits_to_g(float (&x)[32], const ExpFrom<EXACT>& ex, float s, float factor, uint32_t target, uint32_t valid, bool in) {
    float hit = 0.f;
    if (target < 32) {
#pragma unroll
        for (int j = 0; j < 32; j++) hit = target == (uint32_t)j ? x[j] : hit;
        hit = (ex(hit) - s) * factor;
    }
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
        const float2 g = mul2(ex(make_float2(x[j], x[j + 1])), make_float2(factor, factor));
        x[j] = g.x;
        x[j + 1] = g.y;
    }
    if (target < 32) {
#pragma unroll
        for (int j = 0; j < 32; j++) x[j] = target == (uint32_t)j ? hit : x[j];
    }
    if (!in || valid < 32) {
#pragma unroll
        for (int j = 0; j < 32; j++)
            if (!in || j >= (int)valid) x[j] = 0.f;
    }
}
// Two values as 16-bit ones, rounded; with `more`, they are left as what the rounding leaves (nothing of an infinity or a NaN).
template <typename S>
__device__ __forceinline__ uint32_t next_part(float& lo, float& hi, bool more) {
    const uint32_t w = pack2<S>(lo, hi);
    if (more) {
        const float2 got = unpack2<S>(w);
        lo = isfinite(lo) ? lo - got.x : 0.f;
        hi = isfinite(hi) ? hi - got.y : 0.f;
    }
    return w;
}
// What a scored row brings to its line of G.
struct RowOfG {
    uint32_t target;
    float m, s, factor;
    __device__ __forceinline__ RowOfG(const ProductArgs& a, uint32_t slot) {
        const uint32_t row = (uint32_t)a.row_of[slot];
        const float2 st = a.stats[row];
        target = (uint32_t)a.targets[row];
        m = st.x;
        s = st.y;
        factor = (a.mask ? a.mask[row] : 1.f) * a.meta->up / s;
    }
    __device__ __forceinline__ RowOfG() : target(0xffffffffu), m(0.f), s(1.f), factor(0.f) {}
};

// T: type of the operands, S: type of the parts they come in, G: type of d_weight; PARTS: parts of G
template <typename T, typename S, typename G, int P, int PARTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MMA_THREADS, 1)
    k_head_product(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_shares, const ProductArgs a) {
    constexpr bool A_LINES = P == D_WEIGHT, B_LINES = P == D_HIDDEN || P == D_WEIGHT, LOGITS = P == LOGITS_STATS || P == LOGITS_GRAD;
    constexpr bool F32 = sizeof(T) == 4;
    // steps of K that stay in an accumulator (0: all): see above. f32 operands add 6 products of 64 a step, the five small ones first;
    // d_hidden and d_weight in 16 bits hide the cut. 16-bit logits of up to WHOLE steps stay in one: what they lose is small (8e-8 of the
    // loss at hidden 384, 5e-8 by runs), and a way out more would cost the batch 4 % (8191 x 384 x 32000)
    constexpr uint32_t RUN = F32 ? 2 : LOGITS || (P == D_WEIGHT && sizeof(G) == 4) ? 4 : 0, WHOLE = LOGITS && !F32 ? 8 : 0;
    auto run_of = [](uint32_t steps) { return RUN == 0 || steps <= WHOLE ? steps : RUN; };
    extern __shared__ __align__(16) unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
    const uint32_t bars = base + STAGES * STAGE_BYTES + EPILOGUE_WARPS * OUT_BYTES;
    auto full = [&](uint32_t i) { return bars + 8 * i; };
    auto empty = [&](uint32_t i) { return bars + 8 * (STAGES + i); };
    auto done = [&](uint32_t i) { return bars + 8 * (2 * STAGES + i); };       // a run is in accumulator buffer i
    auto taken = [&](uint32_t i) { return bars + 8 * (2 * STAGES + 2 + i); };  // ... and has been read out by both blocks
    __shared__ uint32_t tmem_at, dead;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, rank = cluster_rank();
    const WaitState ws{&dead, a.expired};

    if (threadIdx.x == 0) {
        dead = 0;
        for (int i = 0; i < STAGES; i++) {
            mbar_init(full(i), 1);
            mbar_init(empty(i), 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(done(i), 1);
            mbar_init(taken(i), 2 * EPILOGUE_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch_map(&map_a);
        tma_prefetch_map(&map_b);
        tma_prefetch_map(&map_out);
    }
    if (warp == 1) tmem_alloc_pair(smem_u32(&tmem_at), 512);
    fence_before_sync();
    __syncthreads();
    cluster_sync();
    fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&tmem_at);
    if (!a.beside) after_previous();
    let_next();

    const uint32_t n = a.meta->n;
    const uint32_t M = P == D_WEIGHT ? a.columns : n, N = LOGITS ? a.columns : a.hidden;
    const uint32_t K = P == D_HIDDEN ? a.columns : P == D_WEIGHT ? n : a.hidden;
    const uint32_t wide = LOGITS ? a.width : MMA_N;
    const uint32_t mt = tiles_of(M, MMA_M), nt = tiles_of(N, wide), steps = tiles_of(K, MMA_K);
    const bool skip = P == LOGITS_GRAD && a.keep && a.meta->kept;  // k_head_grad_kept has made G from the logits that are kept
    const Split split(n, a.hidden, a.piece, gridDim.x / 2, min_share(sizeof(T)));
    struct Tile {
        uint32_t m0, n0, width, half, k0, steps, share;
    };
    const uint32_t items = P == D_HIDDEN ? split.items() : skip ? 0 : mt * nt, pairs = gridDim.x / 2;
    auto tile_at = [&](uint32_t t) {
        Tile r;
        uint32_t m, c;
        r.k0 = 0;
        r.steps = steps;
        r.share = 0;
        if (P == D_HIDDEN && t >= split.whole) {
            const uint32_t q = t - split.whole;
            r.share = q / split.rest;
            t = split.whole + (q - r.share * split.rest);
            r.k0 = (uint32_t)((uint64_t)steps * r.share / split.shares);
            r.steps = (uint32_t)((uint64_t)steps * (r.share + 1) / split.shares) - r.k0;
        }
        if (LOGITS) {  // the rows run fastest: one stretch of W serves them all
            m = t % mt;
            c = t / mt;
        } else {
            c = t % nt;
            m = t / nt;
        }
        r.m0 = m * MMA_M;
        r.n0 = c * wide;
        r.width = min(wide, (N - r.n0 + 31) & ~31u);
        r.half = r.width / 2;
        return r;
    };

    if (warp == 0 && lane == 0) {
        // ---- loads
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t t = blockIdx.x / 2; t < items && ok; t += pairs) {
            const Tile c = tile_at(t);
            const uint32_t b_boxes = c.half > 64 ? 2 : 1, run = run_of(c.steps);
            for (uint32_t k1 = 0; k1 < c.steps && ok; k1 += run) {
                for (uint32_t p = 0; p < (uint32_t)a.n_pairs && ok; p++) {
                    const int32_t za = a.pair_a[p], zb = a.pair_b[p];
                    for (uint32_t k = k1; k < min(k1 + run, c.steps); k++, it++) {
                        const uint32_t st = it % STAGES, use = it / STAGES;
                        if (!(ok = mbar_wait(empty(st), (use & 1) ^ 1, ws))) break;
                        const uint32_t to = base + st * STAGE_BYTES, bar = peer_smem(full(st), 0);
                        if (rank == 0) mbar_expect(full(st), 2 * (2 + b_boxes) * BOX_BYTES);
                        const int32_t kk = (int32_t)(c.k0 + k) * 64, m = (int32_t)(c.m0 + rank * 128);
                        const int32_t bn = (int32_t)(c.n0 + rank * c.half + (LOGITS ? a.first : 0));
                        const int32_t bk = kk + (int32_t)(P == D_HIDDEN ? a.first : 0);
                        for (int i = 0; i < 2; i++) {
                            if (P == D_WEIGHT) tma_load_pair(to + i * BOX_BYTES, &map_a, 0, kk, za * (int32_t)a.g_blocks + m / 64 + i, bar);
                            else if (P == D_HIDDEN) tma_load_pair(to + i * BOX_BYTES, &map_a, 0, m + 64 * i, za * (int32_t)a.g_blocks + kk / 64, bar);
                            else tma_load_pair(to + i * BOX_BYTES, &map_a, kk, m + 64 * i, za, bar);
                        }
                        for (int i = 0; i < (int)b_boxes; i++) {
                            if (B_LINES) tma_load_pair(to + (2 + i) * BOX_BYTES, &map_b, bn + 64 * i, bk, zb, bar);
                            else tma_load_pair(to + (2 + i) * BOX_BYTES, &map_b, bk, bn + 64 * i, zb, bar);
                        }
                    }
                }
            }
        }
        // every stage has been given back before the block ends: no load and no arrival is on its way any more
        for (uint32_t i = 1; i <= min(it, (uint32_t)STAGES) && ok; i++) ok = mbar_wait(empty((it - i) % STAGES), ((it - i) / STAGES) & 1, ws);
        if (!ok)  // a wait ran out: what is in flight lands meanwhile
            for (int i = 0; i < 2000; i++) __nanosleep(1000);
    } else if (warp == 1 && lane == 0 && rank == 0) {
        // ---- products
        uint32_t it = 0, round = 0;
        bool ok = true;
        for (uint32_t t = blockIdx.x / 2; t < items && ok; t += pairs) {
            const Tile c = tile_at(t);
            const uint32_t idesc = instruction(a.bf16, A_LINES, B_LINES, MMA_M, c.width), run = run_of(c.steps);
            for (uint32_t k1 = 0; k1 < c.steps && ok; k1 += run, round++) {
                const uint32_t total = min(run, c.steps - k1) * a.n_pairs, buf = round & 1, d = tmem + buf * 256;
                if (!(ok = mbar_wait(taken(buf), ((round >> 1) & 1) ^ 1, ws))) break;
                fence_after_sync();
                for (uint32_t k = 0; k < total; k++, it++) {
                    const uint32_t st = it % STAGES;
                    if (!(ok = mbar_wait(full(st), (it / STAGES) & 1, ws))) break;
                    fence_after_sync();
                    const uint32_t sa = base + st * STAGE_BYTES, sb = sa + 2 * BOX_BYTES;
#pragma unroll
                    for (int q = 0; q < 4; q++)  // 16 of K: 32 bytes along a line, or 16 lines
                        mma_pair(d, operand(sa + q * (A_LINES ? 2048 : 32), A_LINES), operand(sb + q * (B_LINES ? 2048 : 32), B_LINES), idesc,
                                 k > 0 || q > 0);
                    commit_pair(empty(st));
                }
                commit_pair(done(buf));
            }
        }
    } else if (warp >= 2) {
        // ---- the finished tiles: a warp reads the 32 lanes of its quarter, half of the columns each
        const uint32_t quarter = warp & 3, side = (warp - 2) / 4, row_in = quarter * 32 + lane;
        const uint32_t out_base = base + STAGES * STAGE_BYTES + (warp - 2) * OUT_BYTES;
        uint32_t out_now = 0;  // which of the warp's two buffers the last box left from
        const float scale = P == D_WEIGHT ? a.scale * a.meta->down : 1.f;
        const uint32_t kept = P == LOGITS_STATS && a.keep ? a.meta->kept : 0;
        uint32_t round = 0;
        bool ok = true;
        // what a tile's rows need is fetched a tile ahead
        RowOfG next_row;
        auto fetch_row = [&](uint32_t t) {
            if (!LOGITS || t >= items) return;
            const uint32_t i = (t % mt) * MMA_M + rank * 128 + row_in;
            if (i >= M) next_row = RowOfG();
            else if (P == LOGITS_GRAD) next_row = RowOfG(a, i);
            else next_row.target = (uint32_t)a.targets[a.row_of[i]];
        };
        fetch_row(blockIdx.x / 2);
        for (uint32_t t = blockIdx.x / 2; t < items && ok; t += pairs) {
            const Tile c = tile_at(t);
            const uint32_t i = c.m0 + rank * 128 + row_in;
            const bool in = i < M;
            const RowOfG row = next_row;
            fetch_row(t + pairs);
            // column of the tile that the target has; far outside it where another tile has it
            const uint32_t target = LOGITS && in ? row.target - a.first - c.n0 : 0xffffffffu;
            const ExpFrom<F32> ex(row.m);
            const uint32_t valid = min(wide, N - c.n0);  // columns of the tile that exist
            const uint32_t from = side * (wide / 2), to = min(from + wide / 2, P == LOGITS_GRAD ? (valid + 63) & ~63u : valid);
            // the tile's 128 columns of this warp leave tensor memory at once, which frees the accumulator for the next tile
            float acc[4][32];
            auto run_done = [&]() {  // a run is in the accumulator buffer
                ok = __all_sync(0xffffffffu, mbar_wait(done(round & 1), (round >> 1) & 1, ws));
                fence_after_sync();
                return tmem + (round & 1) * 256 + from + (quarter << 21);
            };
            auto run_taken = [&]() {
                fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_peer(peer_smem(taken(round & 1), 0));
                round++;
            };
            if (LOGITS || c.steps) {
                // columns past the tile's width hold what an earlier tile left, and are not used
                const uint32_t at = run_done();
                if (!ok) break;
#pragma unroll
                for (int q = 0; q < 4; q++) tmem_load(at + 32 * q, acc[q]);
                tmem_wait();
#pragma unroll
                for (int q = 0; q < 4; q++) arrived(acc[q]);
                run_taken();
            } else {  // no scored row: a sum of nothing
#pragma unroll
                for (int q = 0; q < 4; q++)
#pragma unroll
                    for (int j = 0; j < 32; j++) acc[q][j] = 0.f;
            }
            if constexpr (RUN > 0) {
                for (uint32_t k1 = run_of(c.steps); k1 < c.steps; k1 += RUN) {
                    const uint32_t at = run_done();
                    if (!ok) break;
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        float x[16];
                        tmem_load(at + 16 * e, x);
                        tmem_wait();
                        arrived(x);
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            float* to = &acc[e / 2][16 * (e & 1) + j];
                            const float2 sum = add2(make_float2(to[0], to[1]), make_float2(x[j], x[j + 1]));
                            to[0] = sum.x;
                            to[1] = sum.y;
                        }
                    }
                    run_taken();
                }
                if (!ok) break;
            }
            const int32_t line = (int32_t)(c.m0 + rank * 128 + quarter * 32);  // the warp's first row
            // lines of the logits that no product reads: d_weight reads G up to the next step of K, and d_hidden's lines past the last
            // scored row are not read themselves
            const bool idle = LOGITS && (uint32_t)line >= (P == LOGITS_GRAD ? (n + 63) & ~63u : n);
            // 128 bytes of each of the warp's rows go out as one box: 16-byte pieces in the order of the 128-byte swizzle, no two lanes of
            // a quarter warp in one bank
            auto box = [&](const CUtensorMap& map, int32_t x, int32_t y, int32_t z, const uint32_t (&w)[32], bool add) {
                if (lane == 0) store_read<1>();
                __syncwarp();
                out_now ^= OUT_BYTES / 2;
                const uint32_t out_at = out_base + out_now;
#pragma unroll
                for (int p = 0; p < 8; p++) st_shared16(out_at + lane * 128 + ((p ^ (lane & 7)) << 4), w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]);
                store_fence();
                __syncwarp();
                if (lane == 0) {
                    if (add) tma_add(&map, x, y, z, out_at);
                    else tma_store(&map, x, y, z, out_at);
                }
            };
            auto words = [&](int q, uint32_t (&w)[32]) {
#pragma unroll
                for (int j = 0; j < 32; j++) w[j] = __float_as_uint(acc[q][j]);
            };
            if constexpr (P == LOGITS_STATS) {
                float m8[8];
#pragma unroll
                for (int k = 0; k < 8; k++) m8[k] = -INFINITY;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint32_t c0 = from + 32 * q;
                    if (c0 >= to || idle) break;
                    if (kept) {
                        uint32_t w[32];
                        words(q, w);
                        box(map_out, (int32_t)(c.n0 + c0), line, 0, w, false);
                    }
                    if (target - c0 < 32) {
                        float tl = 0.f;
#pragma unroll
                        for (int j = 0; j < 32; j++) tl = target - c0 == (uint32_t)j ? acc[q][j] : tl;
                        a.target_logit[i] = tl;
                    }
                    if (c0 + 32 > to) {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (c0 + j >= to) acc[q][j] = -INFINITY;  // no word of the vocabulary
                    }
#pragma unroll
                    for (int j = 0; j < 32; j++) m8[j & 7] = fmaxf(m8[j & 7], acc[q][j]);
                }
                // eight sums side by side: the chains, not the instructions, are what a tile waits for
                const float m = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])), fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7])));
                const ExpFrom<F32> e(m == -INFINITY ? 0.f : m);  // nothing above -inf: exp(-inf - 0) is the zero it should be
                float2 s4[4];
#pragma unroll
                for (int k = 0; k < 4; k++) s4[k] = make_float2(0.f, 0.f);
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    if (from + 32 * q >= to || idle) break;
#pragma unroll
                    for (int j = 0; j < 32; j += 2) s4[j / 2 & 3] = add2(s4[j / 2 & 3], e(make_float2(acc[q][j], acc[q][j + 1])));
                }
                const float2 s1 = add2(add2(s4[0], s4[1]), add2(s4[2], s4[3])), run_stats = make_float2(m, s1.x + s1.y);
                if (in) a.part[(uint64_t)(2 * (c.n0 / wide) + side) * a.pitch + i] = run_stats;
            } else if constexpr (P == LOGITS_GRAD) {
#pragma unroll
                for (int q = 0; q < 4; q += 2) {
                    const uint32_t c0 = from + 32 * q;
                    if (c0 >= to || idle) break;
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        logits_to_g(acc[q + e], ex, row.s, row.factor, target - c0 - 32 * e, valid - min(valid, c0 + 32 * e), in);
#pragma unroll
                    for (int p = 0; p < PARTS; p++) {
                        uint32_t w[32];
#pragma unroll
                        for (int j = 0; j < 32; j++) w[j] = next_part<S>(acc[q + j / 16][2 * (j & 15)], acc[q + j / 16][2 * (j & 15) + 1], p + 1 < PARTS);
                        box(map_out, 0, line, (int32_t)(p * a.g_blocks + (c.n0 + c0) / 64), w, false);
                    }
                }
            } else if constexpr (P == D_HIDDEN) {
                // shares after the first are tiles of their own
                const uint32_t tile = (c.share - 1) * split.rest + (c.m0 / MMA_M * nt + c.n0 / MMA_N) - split.whole;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint32_t c0 = from + 32 * q;
                    if (c0 >= to) break;
                    uint32_t w[32];
                    words(q, w);
                    if (c.share == 0) box(map_out, (int32_t)(c.n0 + c0), line, 0, w, a.add);
                    else box(map_shares, (int32_t)c0, (int32_t)(tile * MMA_M + (line - c.m0)), 0, w, a.add);
                }
            } else if (a.boxes) {
                constexpr int PER = 4 / (int)sizeof(G);  // spans of 32 columns in a box
#pragma unroll
                for (int q = 0; q < 4; q += PER) {
                    const uint32_t c0 = from + 32 * q;
                    if (c0 >= to) break;
                    uint32_t w[32];
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        if constexpr (sizeof(G) == 4) w[j] = __float_as_uint(acc[q][j] * scale);
                        else w[j] = pack2<G>(acc[q + j / 16][2 * (j & 15)] * scale, acc[q + j / 16][2 * (j & 15) + 1] * scale);
                    }
                    box(map_out, (int32_t)(c.n0 + c0), (int32_t)a.first + line, 0, w, sizeof(G) == 4 && a.accumulate);
                }
            } else {
                // 16-bit sums with what was there, or rows that are not whole 16-byte pieces: 32 x 32 results are turned in shared memory, so
                // that a warp writes 32 neighbours
                const uint32_t rows = min(32u, M - min(M, (uint32_t)line));
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    const uint32_t c0 = from + 32 * q;
                    if (c0 >= to) break;
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        const uint32_t at = out_base + lane * 128 + ((j ^ lane) << 2);
                        asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(acc[q][j] * scale) : "memory");
                    }
                    __syncwarp();
                    G* out = static_cast<G*>(a.dw) + (uint64_t)(a.first + line) * a.hidden + c.n0 + c0 + lane;
                    const bool here = c0 + lane < valid;
#pragma unroll 8
                    for (uint32_t k = 0; k < rows; k++, out += a.hidden) {
                        float v;
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(out_base + k * 128 + ((lane ^ k) << 2)) : "memory");
                        if (here) *out = from_f32<G>(a.accumulate ? to_f32<G>(*out) + v : v);
                    }
                }
            }
        }
        if (lane == 0) store_done();
    }
    __syncwarp();
    fence_before_sync();
    __syncthreads();
    cluster_sync();  // nobody arrives at a barrier of a block that has ended
    fence_after_sync();
    if (warp == 1) tmem_free_pair(tmem, 512);
    if (a.beside) after_previous();
}

// ---- a piece of G from logits that the losses have kept, the same bits as the product would give. A thread takes 32 columns of a
// scored row; the rows up to the next step of d_weight's K are zeros.
template <typename T, typename S, int PARTS>
__global__ void __launch_bounds__(256) k_head_grad_kept(const ProductArgs a) {
    let_next();
    after_previous();
    const uint32_t n = a.meta->n, kept = a.meta->kept;
    if (kept == 0 || n == 0) return;
    const uint32_t per = ((a.columns + 63) & ~63u) / 32;
    const uint64_t total = (uint64_t)((n + 63) & ~63u) * per;
    for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (uint64_t)gridDim.x * 256) {
        const uint32_t slot = (uint32_t)(e / per), c0 = (uint32_t)(e - (uint64_t)slot * per) * 32;
        const bool in = slot < n;
        RowOfG row;
        float g[32];
        if (in) {
            row = RowOfG(a, slot);
            const float* from = a.l + (uint64_t)slot * kept + a.first + c0;
#pragma unroll
            for (int q = 0; q < 4; q++) load32(from + 8 * q, reinterpret_cast<uint32_t*>(g) + 8 * q);
        } else {
#pragma unroll
            for (int j = 0; j < 32; j++) g[j] = 0.f;
        }
        const ExpFrom<sizeof(T) == 4> ex(row.m);
        logits_to_g(g, ex, row.s, row.factor, in ? row.target - a.first - c0 : 0xffffffffu, a.columns - min(a.columns, c0), in);
#pragma unroll
        for (int p = 0; p < PARTS; p++) {
            S* out = static_cast<S*>(a.g) + ((uint64_t)(p * a.g_blocks + c0 / 64) * a.cap + slot) * 64 + c0 % 64;
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; j++) w[j] = next_part<S>(g[2 * j], g[2 * j + 1], p + 1 < PARTS);
            store32(out, w);
            store32(out + 16, w + 8);
        }
    }
}

// ---- d_hidden: the scored rows' sums, their shares in order, times the scale, rounded; zeros for the others
// N columns a thread: four, so that a small d_hidden spreads over the SMs, or one where rows are not aligned. GROUPS warps of a block
// share the shares of 32 x N elements, in order, and are joined in order: a small d_hidden has many shares and few elements, and a thread
// alone would wait for one load after the other (122 x 128, 73 shares: 15 us, 6 in 8 groups).
template <typename T, int N, int GROUPS>
__global__ void __launch_bounds__(256) k_head_d_hidden(uint32_t rows, uint32_t hidden, uint32_t dx_pitch, uint64_t piece, uint32_t pairs,
                                                       const int32_t* __restrict__ slot_of, const float* __restrict__ dx,
                                                       const float* __restrict__ dx_shares, const HeadMeta* __restrict__ meta, float scale, T* out,
                                                       uint64_t stride) {
    static_assert(GROUPS == 1 || GROUPS == 8, "warps of a block");
    __shared__ float joined[GROUPS > 1 ? 8 : 1][32 * N];
    let_next();
    after_previous();
    scale *= meta->down;
    const Split split(meta->n, hidden, piece, pairs, min_share(sizeof(T)));
    const uint32_t per = (hidden + N - 1) / N, nt = tiles_of(hidden, MMA_N), group = GROUPS > 1 ? threadIdx.x / 32 : 0;
    const uint64_t total = (uint64_t)rows * per;
    constexpr uint32_t AT_ONCE = 256 / GROUPS;  // elements of N columns a block takes
    for (uint64_t e0 = (uint64_t)blockIdx.x * AT_ONCE; e0 < total; e0 += (uint64_t)gridDim.x * AT_ONCE) {
        const uint64_t e = e0 + threadIdx.x % AT_ONCE;
        const bool here = e < total;
        const uint32_t row = here ? (uint32_t)(e / per) : 0, col = here ? (uint32_t)(e - (uint64_t)row * per) * N : 0;
        const int32_t slot = here ? slot_of[row] : -1;
        Vec<float, N> sum;
#pragma unroll
        for (int j = 0; j < N; j++) sum.e[j] = 0.f;
        if (slot >= 0) {
            const uint32_t tile = slot / MMA_M * nt + col / MMA_N;
            const float* from = dx_shares + ((uint64_t)tile - split.whole) * (MMA_M * MMA_N) + slot % MMA_M * MMA_N + col % MMA_N;
            const uint32_t shares = tile >= split.whole ? split.shares : 1, each = (shares + GROUPS - 1) / GROUPS;
            uint32_t k = group * each;
            const uint32_t end = min(shares, k + each);
            if (k == 0) {
                sum.load(dx + (uint64_t)slot * dx_pitch + col);
                k = 1;
            }
            constexpr int AHEAD = 8;
            for (; k < end; k += AHEAD) {
                Vec<float, N> v[AHEAD];
#pragma unroll
                for (int a = 0; a < AHEAD; a++)
                    if (k + a < end) v[a].load(from + (uint64_t)(k + a - 1) * split.rest * (MMA_M * MMA_N));
#pragma unroll
                for (int a = 0; a < AHEAD; a++)
                    if (k + a < end) {
#pragma unroll
                        for (int j = 0; j < N; j++) sum.e[j] += v[a].e[j];
                    }
            }
        }
        if constexpr (GROUPS > 1) {
            __syncthreads();  // the sums of the round before have been read
#pragma unroll
            for (int j = 0; j < N; j++) joined[group][threadIdx.x % 32 + 32 * j] = sum.e[j];
            __syncthreads();
            if (group) continue;
            for (int g = 1; g < GROUPS; g++)
#pragma unroll
                for (int j = 0; j < N; j++) sum.e[j] += joined[g][threadIdx.x + 32 * j];
        }
        if (!here) continue;
        Vec<T, N> o;
#pragma unroll
        for (int j = 0; j < N; j++) o.e[j] = from_f32<T>(slot < 0 ? 0.f : sum.e[j] * scale);
        o.store(out + (uint64_t)row * stride + col);
    }
}

bool misaligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) % to) != 0; }

using Encode = decltype(&cuTensorMapEncodeTiled);
int32_t encoder(Encode* out) {
    static std::atomic<Encode> found{nullptr};  // handles of several threads ask; whoever comes first finds the same
    Encode fn = found.load(std::memory_order_acquire);
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult st;
        OXZ_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &st));
        if (st != cudaDriverEntryPointSuccess || !p) return fail(OXZ_ERR_UNSUPPORTED, "the driver has no cuTensorMapEncodeTiled");
        fn = reinterpret_cast<Encode>(p);
        found.store(fn, std::memory_order_release);
    }
    *out = fn;
    return OXZ_OK;
}

// [parts][lines][pitch] values as boxes of 128 bytes by `box_lines`, 128-byte swizzle; what lies outside reads as zeros and is not written
int32_t tensor_map(CUtensorMap* m, int32_t dtype, const void* base, uint64_t pitch, uint64_t lines, uint64_t parts, uint64_t part_stride,
                   uint32_t box_lines = 64) {
    Encode encode = nullptr;
    OXZ_TRY(encoder(&encode));
    const uint32_t es = (uint32_t)dtype_size(dtype);
    const cuuint64_t dims[3] = {pitch, lines, parts}, strides[2] = {pitch * es, part_stride * es};
    const cuuint32_t box[3] = {128 / es, box_lines, 1}, step[3] = {1, 1, 1};
    const CUtensorMapDataType t = dtype == OXZ_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == OXZ_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const CUresult r = encode(m, t, 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(OXZ_ERR_CUDA, "cuTensorMapEncodeTiled failed: %d", (int)r);
    return OXZ_OK;
}

// Width of the logits' tiles: halved while all of them still run at once (the losses of 149 x 1088 x 2918 f32: 61 us with 12 tiles of 256
// columns, 54 with 46 of 64). To fill the last of several rounds it does not pay, since a narrow tile loads as much of X as a wide one
// (2048 x 2048 x 2500 bf16: 43 us with 80 tiles of 256, 51 with 160 of 128).
uint32_t tile_width(const oxz_head* h, uint64_t rows, uint64_t columns, uint32_t least) {
    uint32_t w = MMA_N;
    while (w > least && (uint64_t)tiles_of(rows, MMA_M) * tiles_of(columns, w / 2) <= (uint64_t)h->clusters) w /= 2;
    return w;
}

template <typename T, typename S, typename G, int PARTS>
struct Products {
    template <int P>
    static int32_t launch(const oxz_head* h, const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& out, const CUtensorMap& shares,
                          const ProductArgs& a, uint64_t m, uint64_t n, cudaStream_t s) {
        const uint64_t tiles = (uint64_t)tiles_of(m, MMA_M) * tiles_of(n, P == LOGITS_STATS || P == LOGITS_GRAD ? a.width : MMA_N);
        // the cut of D_HIDDEN goes by the number of pairs: always all of them
        const unsigned pairs = P == D_HIDDEN ? (unsigned)h->clusters : (unsigned)std::min<uint64_t>(tiles, h->clusters);
        if (tiles) OXZ_CUDA(launch_after(true, k_head_product<T, S, G, P, PARTS>, 2 * pairs, MMA_THREADS, MMA_SMEM, s, ma, mb, out, shares, a));
        return OXZ_OK;
    }
    template <int P>
    static int32_t prepare(int* clusters) {
        auto k = k_head_product<T, S, G, P, PARTS>;
        OXZ_CUDA(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MMA_SMEM));
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(2);
        cfg.blockDim = dim3(MMA_THREADS);
        cfg.dynamicSmemBytes = MMA_SMEM;
        cudaLaunchAttribute attr{};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim = {2, 1, 1};
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int c = 0;
        OXZ_CUDA(cudaOccupancyMaxActiveClusters(&c, k, &cfg));
        if (c < 1) return fail(OXZ_ERR_UNSUPPORTED, "the device runs no pair of blocks with %u bytes of shared memory", MMA_SMEM);
        *clusters = *clusters ? std::min(*clusters, c) : c;
        return OXZ_OK;
    }
    static int32_t prepare_all(oxz_head* h) {
        OXZ_TRY(prepare<LOGITS_STATS>(&h->clusters));
        OXZ_TRY(prepare<LOGITS_GRAD>(&h->clusters));
        OXZ_TRY(prepare<D_HIDDEN>(&h->clusters));
        OXZ_TRY(prepare<D_WEIGHT>(&h->clusters));
        return few_prepare<T, G>();
    }

    // A handful of rows: see oxz_head_few.cuh
    static int32_t run_few(oxz_head* h, const oxz_head_batch& b, bool wide, float* row_loss, float2* row_stats, bool want_loss, float* totals,
                           const oxz_head_grads* gr, cudaStream_t s) {
        const oxz_head_desc& d = h->d;
        FewArgs a{};
        a.x = b.hidden;
        a.x_stride = b.hidden_stride;
        a.w = b.weight;
        a.targets = b.targets;
        a.mask = b.loss_mask;
        a.rows = (uint32_t)b.rows;
        a.hidden = (uint32_t)d.hidden;
        a.vocab = (uint32_t)d.vocab;
        a.logits = h->few_logits;
        a.part = h->few_part;
        a.done = h->few_done;
        a.stats = row_stats ? row_stats : h->stats;
        a.row_loss = row_loss;
        a.totals = totals;
        a.finish = want_loss;
        bool out_wide = true;
        if (gr) {
            a.dw = gr->d_weight;
            a.dx = gr->d_hidden;
            a.dx_stride = gr->d_hidden_stride;
            a.dx_part = h->few_dx;
            a.scale = (float)gr->grad_scale;
            a.accumulate = gr->accumulate && gr->d_weight;
            a.want_dx = gr->d_hidden != nullptr;
            out_wide = d.hidden % 4 == 0;  // weight and d_weight begin on 16 bytes; x is read by elements
        }
        return few_run<T, G>(a, wide, out_wide, gr != nullptr, h->sms, s);
    }

    static int32_t run(oxz_head* h, const oxz_head_batch& b, float* row_loss, float2* row_stats, bool want_loss, float* totals,
                       const oxz_head_grads* gr, cudaStream_t s) {
        const oxz_head_desc& d = h->d;
        const bool on16 = !misaligned(b.hidden, 16) && b.hidden_stride * sizeof(T) % 16 == 0 && d.hidden * sizeof(T) % 16 == 0;
        if (few_fits(b.rows, d.hidden, d.vocab, sizeof(T), on16))
            return run_few(h, b, on16, row_loss, row_stats, want_loss, totals, gr, s);
        constexpr bool F32 = sizeof(T) == 4, BF16 = std::is_same<S, __nv_bfloat16>::value;
        const size_t es = sizeof(T);
        const unsigned many = (unsigned)h->clusters * 2 * 8;  // blocks of the elementwise kernels
        const bool sure = b.rows * h->kept_pitch <= h->l_elems;  // all logits fit, whatever the mask
        const bool keep = want_loss && gr && h->l_elems && (sure || h->keep_large);
        const uint64_t x_part = h->cap * h->pitch, w_part = d.vocab * h->pitch, l_elems = keep ? h->l_elems : 0;
        const bool x_wide = !misaligned(b.hidden, 16) && b.hidden_stride * es % 16 == 0;
        const T* x = static_cast<const T*>(b.hidden);
        const uint64_t pack = (b.rows + MMA_M) * (h->pitch / 8);  // 16-byte pieces at most
        if (b.rows <= LISTED) {
            OXZ_CUDA(launch_after(false, k_head_list_pack<T, S>, (unsigned)std::min<uint64_t>((pack + LISTED - 1) / LISTED, h->sms), LISTED, 0, s, b.targets,
                                  b.loss_mask, (uint32_t)b.rows, d.vocab, h->row_of, h->slot_of, h->meta, !BF16, l_elems, x, b.hidden_stride,
                                  (uint32_t)d.hidden, h->pitch, static_cast<S*>(h->x), x_part, h->parts, x_wide));
        } else {
            OXZ_CUDA(launch_after(false, k_head_rows, 1, 1024, 0, s, b.targets, b.loss_mask, (uint32_t)b.rows, d.vocab, h->row_of, h->slot_of, h->meta, !BF16,
                                  l_elems));
            OXZ_CUDA(launch_after(true, k_head_pack<T, S>, (unsigned)std::min<uint64_t>((pack + 255) / 256, many), 256, 0, s, x, b.hidden_stride,
                                  (uint32_t)d.hidden, h->pitch, b.rows, h->row_of, h->meta, static_cast<S*>(h->x), x_part, h->parts, x_wide));
        }
        if (h->w)
            OXZ_CUDA(launch_after(true, k_head_pack<T, S>, many, 256, 0, s, static_cast<const T*>(b.weight), d.hidden, (uint32_t)d.hidden, h->pitch, d.vocab,
                                  nullptr, h->meta, static_cast<S*>(h->w), w_part, h->parts, d.hidden * es % 16 == 0));
        constexpr int32_t ST = BF16 ? OXZ_BF16 : OXZ_F16;
        CUtensorMap mx, mw, mg;
        OXZ_TRY(tensor_map(&mx, ST, h->x, h->pitch, h->cap, h->parts, x_part));
        OXZ_TRY(tensor_map(&mw, ST, h->w ? h->w : b.weight, h->pitch, d.vocab, h->parts, w_part));

        ProductArgs a{};
        a.meta = h->meta;
        a.row_of = h->row_of;
        a.hidden = (uint32_t)d.hidden;
        a.pitch = (uint32_t)b.rows;
        a.dx_pitch = h->dx_pitch;
        a.targets = b.targets;
        a.mask = b.loss_mask;
        a.part = h->part;
        a.target_logit = h->target_logit;
        a.g = h->g;
        a.dx = h->dx;
        a.l = h->l;
        a.bf16 = BF16;
        a.dx_shares = h->dx_shares;
        a.piece = (uint32_t)h->piece;
        a.keep = keep;
        a.expired = h->d_expired;
        // an f32 operand is hi + mid + lo; of the nine products the six above 2^-24 are formed, the small ones first
        static const uint8_t six[2][6] = {{2, 1, 0, 1, 0, 0}, {0, 1, 2, 0, 1, 0}};
        auto pairs = [&](int g_only) {
            a.n_pairs = F32 ? 6 : g_only;
            for (int p = 0; p < a.n_pairs; p++) {
                a.pair_a[p] = F32 ? six[0][p] : (uint8_t)(g_only - 1 - p);
                a.pair_b[p] = F32 ? six[1][p] : 0;
            }
        };
        float2* stats = row_stats ? row_stats : h->stats;
        pairs(1);
        if (want_loss) {
            a.columns = (uint32_t)d.vocab;
            a.width = tile_width(h, b.rows, d.vocab, 64);
            CUtensorMap ml = mx;  // not used where nothing is kept
            if (a.keep) OXZ_TRY(tensor_map(&ml, OXZ_F32, h->l, h->kept_pitch, h->l_elems / h->kept_pitch, 1, h->l_elems / h->kept_pitch * h->kept_pitch, 32));
            OXZ_TRY(launch<LOGITS_STATS>(h, mx, mw, ml, ml, a, b.rows, d.vocab, s));
            const bool many_rows = b.rows > (uint64_t)h->sms * FINISH_ROWS / 2;
            const unsigned per = many_rows ? 32 : FINISH_ROWS, blocks = std::max<unsigned>(1, (unsigned)((b.rows + per - 1) / per)), halves = 2 * tiles_of(d.vocab, a.width);
            const unsigned threads = many_rows ? 1024 : std::min(1024u, std::max(256u, (halves / 4 * per + 255) / 256 * 256));
            OXZ_CUDA(launch_after(true, many_rows ? k_head_finish<32> : k_head_finish<FINISH_ROWS>, blocks, threads, 0, s, (uint32_t)b.rows, a.pitch, halves, h->slot_of, h->part,
                                  h->target_logit, b.loss_mask, stats, row_loss, h->loss_part, h->meta, totals));
        }
        if (!gr) return OXZ_OK;
        a.stats = stats;
        a.scale = (float)gr->grad_scale;
        a.accumulate = gr->accumulate;
        a.dw = gr->d_weight;
        a.g_blocks = (uint32_t)(h->piece / 64);
        a.cap = (uint32_t)h->cap;
        OXZ_TRY(tensor_map(&mg, ST, h->g, 64, h->cap, h->piece / 64 * h->g_parts, h->cap * 64));
        CUtensorMap mgo, mdx, mds, mdw = mg;
        OXZ_TRY(tensor_map(&mgo, ST, h->g, 64, h->cap, h->piece / 64 * h->g_parts, h->cap * 64, 32));
        OXZ_TRY(tensor_map(&mdx, OXZ_F32, h->dx, h->dx_pitch, h->cap, 1, h->cap * h->dx_pitch, 32));
        const uint64_t share_lines = (uint64_t)MAX_ROUNDS * h->clusters * MMA_M;
        OXZ_TRY(tensor_map(&mds, OXZ_F32, h->dx_shares, MMA_N, share_lines, 1, share_lines * MMA_N, 32));
        // d_weight leaves by TMA where its rows are whole 16-byte pieces; 16-bit sums with what was there are made by the threads
        a.boxes = gr->d_weight && d.hidden * sizeof(G) % 16 == 0 && (sizeof(G) == 4 || !gr->accumulate);
        if (a.boxes) OXZ_TRY(tensor_map(&mdw, d.grad_dtype, gr->d_weight, d.hidden, d.vocab, 1, d.vocab * d.hidden, 32));
        for (uint64_t v = 0; v < d.vocab; v += h->piece) {
            a.first = (uint32_t)v;
            a.columns = (uint32_t)std::min(h->piece, d.vocab - v);
            a.add = v > 0;
            a.width = tile_width(h, b.rows, a.columns, 128);  // G leaves in boxes of 64 columns
            pairs(1);
            // the scored rows' count decides on the device which of the two has work
            if (a.keep && b.rows) OXZ_CUDA(launch_after(true, k_head_grad_kept<T, S, PARTS>, many, 256, 0, s, a));
            if (!a.keep || !sure) OXZ_TRY(launch<LOGITS_GRAD>(h, mx, mw, mgo, mgo, a, b.rows, a.columns, s));
            if (gr->d_hidden) OXZ_TRY(launch<D_HIDDEN>(h, mg, mw, mdx, mds, a, b.rows, d.hidden, s));
            pairs(h->g_parts);
            a.beside = gr->d_hidden && b.rows;
            if (gr->d_weight) OXZ_TRY(launch<D_WEIGHT>(h, mg, mx, mdw, mdw, a, a.columns, d.hidden, s));
            a.beside = 0;
        }
        if (gr->d_hidden && b.rows) {
            constexpr int N = 4;
            const bool wide = !misaligned(gr->d_hidden, N * es) && gr->d_hidden_stride % N == 0 && d.hidden % N == 0;
            // elements a thread, or a group of eight; eight where they fill the SMs' blocks at most once
            const uint64_t elements = b.rows * ((d.hidden + (wide ? N : 1) - 1) / (wide ? N : 1));
            const bool grouped = elements <= (uint64_t)many * 32;
            auto k = wide ? (grouped ? k_head_d_hidden<T, N, 8> : k_head_d_hidden<T, N, 1>) : (grouped ? k_head_d_hidden<T, 1, 8> : k_head_d_hidden<T, 1, 1>);
            const uint64_t blocks = (elements + (grouped ? 31 : 255)) / (grouped ? 32 : 256);
            OXZ_CUDA(launch_after(true, k, (unsigned)std::min<uint64_t>(blocks, many), 256, 0, s, (uint32_t)b.rows, (uint32_t)d.hidden, h->dx_pitch, h->piece,
                                  (uint32_t)h->clusters, h->slot_of, h->dx, h->dx_shares, h->meta, a.scale,
                                  static_cast<T*>(gr->d_hidden), gr->d_hidden_stride));
        }
        return OXZ_OK;
    }
};
using BF = __nv_bfloat16;
using F32Products = Products<float, BF, float, 3>;
using Bf16Products = Products<BF, BF, BF, 1>;
using Bf16F32Products = Products<BF, BF, float, 3>;
using F16Products = Products<__half, __half, __half, 1>;
using F16F32Products = Products<__half, __half, float, 3>;
// f(P): P the product family of the handle's types
template <typename F>
int32_t with_types(const oxz_head_desc& d, F&& f) {
    if (d.dtype == OXZ_F32) return f(F32Products{});
    if (d.dtype == OXZ_BF16) return d.grad_dtype == OXZ_F32 ? f(Bf16F32Products{}) : f(Bf16Products{});
    return d.grad_dtype == OXZ_F32 ? f(F16F32Products{}) : f(F16Products{});
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
    if (*reinterpret_cast<volatile int32_t*>(h->expired))
        return fail(OXZ_ERR_TIMEOUT, "%s: a bounded wait inside a kernel of an earlier call ran out; its results are not valid", who);
    DeviceGuard dev;
    OXZ_TRY(dev.enter(d.device));
    cudaStream_t s = (cudaStream_t)stream;
    Turn turn(h->order);
    OXZ_TRY(turn.begin(s));
    float2* st = reinterpret_cast<float2*>(row_stats);
    const oxz_head_grads* gp = want_grads ? &g : nullptr;
    const int32_t rc = with_types(d, [&](auto p) { return decltype(p)::run(h, b, row_loss, st, want_loss, totals, gp, s); });
    OXZ_TRY(rc);
    return turn.end();
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
        if (d.max_rows == 0 || d.max_rows > (1ull << 30))
            return fail(OXZ_ERR_INVALID, "oxz_head_create: max_rows %llu is outside 1..2^30", (unsigned long long)d.max_rows);
        if (d.vocab == 0 || d.vocab > (1ull << 30))
            return fail(OXZ_ERR_INVALID, "oxz_head_create: vocab %llu is outside 1..2^30", (unsigned long long)d.vocab);
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
            h->cap = (d.max_rows + MMA_M - 1) / MMA_M * MMA_M;
            h->pitch = (uint32_t)((d.hidden + 7) / 8 * 8);
            h->dx_pitch = (uint32_t)((d.hidden + 31) / 32 * 32);
            h->parts = d.dtype == OXZ_F32 ? 3 : 1;
            h->g_parts = d.grad_dtype == OXZ_F32 ? 3 : 1;
            OXZ_TRY(with_types(d, [&](auto p) { return decltype(p)::prepare_all(h); }));
            OXZ_CUDA(cudaDeviceGetAttribute(&h->sms, cudaDevAttrMultiProcessorCount, d.device));
            // a third of the limit for a piece's G, the rest for logits that are kept, where there are so many
            const uint64_t budget = d.piece_bytes ? d.piece_bytes : 2048ull << 20, limit = budget / 3;
            const uint64_t all = (d.vocab + MMA_N - 1) / MMA_N * MMA_N;
            h->piece = std::min(all, std::max<uint64_t>(MMA_N, limit / (h->cap * 2 * h->g_parts) / MMA_N * MMA_N));
            uint64_t bytes = 0;
            auto get = [&](auto** p, uint64_t n) -> int32_t {  // what a failed attempt left behind is kept and used by the next one
                if (!*p) OXZ_CUDA(cudaMalloc((void**)p, n));
                bytes += n;
                return OXZ_OK;
            };
            OXZ_TRY(get(&h->stats, d.max_rows * 8));
            int few_rows = FEW_ROWS;
            // A handle whose every batch streams the weight never comes to the tiles, and gets none of their workspace
            const bool tiles = !few_always(d.max_rows, d.hidden, d.vocab, dtype_size(d.dtype), &few_rows);
            if (tiles) few_rows = FEW_ROWS;
            h->kept_pitch = all;
            // Kept logits are written and read once (10 bytes of traffic an element with G's 2); forming them again takes 2 x hidden
            // operations on the tensor cores, six times that for f32. Losses with gradients of 2048 rows over 65536 words, bf16, kept
            // and formed again: 579 and 461 us at hidden 384, 839 and 764 at 768, 1033 and 1003 at 1024, 1682 and 1870 at 2048.
            // A batch of few logits keeps them at any width: its time is launches, and G from them takes a light one
            // (100 x 360 x 12300 bf16: 42 us, 48 when they are formed again).
            h->keep_large = d.hidden * (d.dtype == OXZ_F32 ? 6 : 1) >= 1024;
            h->l_elems = std::min(budget / 3 * 2 / 4, std::min<uint64_t>(h->cap * all, h->keep_large ? ~uint64_t(0) : FEW_LOGITS));
            if (h->l_elems < all) h->l_elems = 0;  // not a single row
            if (tiles) {
                OXZ_TRY(get(&h->row_of, d.max_rows * 4));
                OXZ_TRY(get(&h->slot_of, d.max_rows * 4));
                OXZ_TRY(get(&h->part, 2 * std::max<uint64_t>((all / MMA_N) * d.max_rows, (uint64_t)h->clusters * MMA_M) * 8));
                OXZ_TRY(get(&h->target_logit, d.max_rows * 4));
                OXZ_TRY(get(&h->loss_part, (d.max_rows + FINISH_ROWS - 1) / FINISH_ROWS * 8));
                OXZ_TRY(get(&h->meta, sizeof(HeadMeta)));
                OXZ_TRY(get(&h->x, h->cap * h->pitch * h->parts * 2));
                if (d.dtype == OXZ_F32 || d.hidden % 8) OXZ_TRY(get(&h->w, d.vocab * h->pitch * h->parts * 2));
                OXZ_TRY(get(&h->g, h->cap * h->piece * h->g_parts * 2));
                if (h->l_elems) OXZ_TRY(get(&h->l, h->l_elems * 4));
                OXZ_TRY(get(&h->dx, h->cap * h->dx_pitch * 4));
                // rest x shares is at most MAX_ROUNDS x pairs
                OXZ_TRY(get(&h->dx_shares, (uint64_t)MAX_ROUNDS * h->clusters * MMA_M * MMA_N * 4));
            }
            OXZ_TRY(get(&h->few_logits, d.vocab * few_rows * 4));
            OXZ_TRY(get(&h->few_part, (uint64_t)h->sms * FEW_LOGIT_BLOCKS * few_rows * 8));
            OXZ_TRY(get(&h->few_dx, (uint64_t)std::max(few_parts(d.hidden, d.vocab, h->sms, 1), few_parts_16(d.hidden, d.vocab, h->sms)) * few_rows * d.hidden * 4));
            OXZ_TRY(get(&h->few_done, 4));
            OXZ_CUDA(cudaMemset(h->few_done, 0, 4));
            OXZ_CUDA(cudaDeviceSynchronize());
            if (!h->expired) {
                OXZ_CUDA(cudaHostAlloc((void**)&h->expired, 4, cudaHostAllocMapped));
                *h->expired = 0;
                OXZ_CUDA(cudaHostGetDevicePointer((void**)&h->d_expired, h->expired, 0));
            }
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
        if (h->stats) dev.enter(h->d.device);
        h->order.destroy();
        for (void* p : {(void*)h->row_of, (void*)h->slot_of, (void*)h->part, (void*)h->target_logit, (void*)h->stats, (void*)h->loss_part,
                        (void*)h->meta, h->x, h->w, h->g, (void*)h->l, (void*)h->dx, (void*)h->dx_shares, (void*)h->few_logits,
                        (void*)h->few_part, (void*)h->few_dx, (void*)h->few_done})
            if (p) cudaFree(p);
        if (h->expired) cudaFreeHost(h->expired);
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
