// The loss head for a handful of rows, where the products are nothing and the weight's way through the machine is everything: each
// launch streams the weight once, and a batch takes one launch for its losses and two more for its gradients (the tiles of the
// tensor-core path take eight, most of them waits for the one before).
//
//   k_few_logits   logits of all rows for a stretch of the vocabulary, kept as [word][R] in f32; {max, sum} of each row by block, and the
//                  block that ends last joins them in order: statistics, losses, totals
//   k_few_grads    G of a stretch of words from the kept logits, then word by word, a thread holding four columns of every row:
//                  dW[v] = c sum_i G_iv x_i (written), dX_i += G_iv W[v] (registers; a partial sum per block)
//   k_few_d_hidden the blocks' partial sums in order
//
// f32 rows, and 16-bit ones off 16 bytes, are f32 arithmetic in registers, and G is not rounded. 16-bit rows on 16 bytes use the
// 16 x 8 x 16 warp product (mma.sync): at 16 rows the pass is bound by the weight's way, not by the product's rate (128256 words of 2048:
// logits 120 us, 4.4 TB/s; gradients 209 us, 4.85 TB/s). Their gradients take G in two 16-bit parts (k_few_grads_16); an f32 d_weight
// takes k_few_grads and G unrounded. R, the rows a kernel is made for, is 4, 8 or 16.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <algorithm>

#include "oxz_elem.cuh"
#include "oxz_internal.h"

namespace oxz {

constexpr int FEW_ROWS = 16;        // the most rows of this path
constexpr int FEW_THREADS = 256;
constexpr int FEW_WORDS = 64;       // words whose G a block has in shared memory at a time

namespace {

struct FewArgs {
    const void* x;
    uint64_t x_stride;
    const void* w;
    const int64_t* targets;
    const float* mask;
    uint32_t rows, hidden, vocab;
    float* logits;       // [vocab][R]
    float2* part;        // [blocks][R]
    uint32_t* done;      // blocks that have ended; the last puts it back to 0
    float2* stats;       // [rows]
    float* row_loss;     // may be null, as totals
    float* totals;
    int finish;          // join the statistics (0: the caller has them)
    // gradients
    void* dw;
    void* dx;
    uint64_t dx_stride;
    float* dx_part;      // [blocks along the vocabulary][R][hidden]
    uint32_t words;      // a block's stretch of the vocabulary
    float scale;
    int accumulate, want_dx;
};

// A row that takes part: its weight is not zero and its target is a word.
__device__ __forceinline__ bool few_scored(const FewArgs& a, uint32_t i) {
    return i < a.rows && (uint64_t)a.targets[i] < a.vocab && (a.mask == nullptr || a.mask[i] != 0.f);
}

__device__ __forceinline__ float2 join_stats(float2 a, float2 b) {  // {max, sum of exp(x - max)}; an empty set is {-inf, 0}
    const float m = fmaxf(a.x, b.x);
    if (m == -INFINITY) return make_float2(m, a.y + b.y);
    return make_float2(m, a.y * expf(a.x - m) + b.y * expf(b.x - m));
}
__device__ __forceinline__ void add_logit(float2& s, float l) {
    if (l > s.x) {
        s.y = fmaf(s.y, expf(s.x - l), 1.f + (l - l));  // an infinity makes the row NaN, as inf - inf does
        s.x = l;
    } else {
        s.y += l == -INFINITY && s.x == -INFINITY ? 0.f : expf(l - s.x);  // a NaN comes here and stays
    }
}

// The block's rows' sets, one per warp and row in `by_warp`, to part[block]; the last block makes the batch's results of all of them.
template <int R, int WARPS>
__device__ void few_finish(const FewArgs& a, float2 (&by_warp)[WARPS][R]) {
    __shared__ uint32_t last;
    __shared__ double sums[2][R];
    __syncthreads();
    if (threadIdx.x < R) {
        float2 s = by_warp[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < WARPS; w++) s = join_stats(s, by_warp[w][threadIdx.x]);
        a.part[(uint64_t)blockIdx.x * R + threadIdx.x] = s;
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(a.done, 1u) == gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
    // 16 threads a row, each every 16th block, eight at a time
    const uint32_t row = threadIdx.x / 16, k = threadIdx.x & 15;
    float2 s = make_float2(-INFINITY, 0.f);
    if (row < R)
        for (uint32_t b = k; b < gridDim.x; b += 128) {
            float2 p[8];
#pragma unroll
            for (int e = 0; e < 8; e++) p[e] = b + 16 * e < gridDim.x ? __ldcg(&a.part[(uint64_t)(b + 16 * e) * R + row]) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int e = 0; e < 8; e++) s = join_stats(s, p[e]);
        }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) s = join_stats(s, make_float2(__shfl_xor_sync(0xffffffffu, s.x, o), __shfl_xor_sync(0xffffffffu, s.y, o)));
    if (k == 0 && row < R) {
        double loss = 0.0, weight = 0.0;
        if (row < a.rows) {
            const bool on = few_scored(a, row);
            float l = 0.f;
            if (on) {
                l = logf(s.y) - (__ldcg(&a.logits[(uint64_t)a.targets[row] * R + row]) - s.x);
                weight = a.mask ? (double)a.mask[row] : 1.0;
                loss = weight * (double)l;
            }
            a.stats[row] = on ? s : make_float2(0.f, 0.f);
            if (a.row_loss) a.row_loss[row] = l;
        }
        sums[0][row] = loss;
        sums[1][row] = weight;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        if (a.totals) {
            double l = 0.0, w = 0.0;
            for (int i = 0; i < R; i++) {
                l += sums[0][i];
                w += sums[1][i];
            }
            a.totals[0] = (float)l;
            a.totals[1] = (float)w;
        }
        *a.done = 0;
    }
}

__device__ __forceinline__ uint32_t smem_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T>
__device__ __forceinline__ void warp_product(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2) {
        if constexpr (__is_same(T, __nv_bfloat16))
            asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                         : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
        else
            asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                         : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// 16-bit logits, rows on 16 bytes. A warp takes 16 words. Lane (r, q) = (lane / 4, lane % 4) has 16 bytes, elements 8q .. 8q + 7 of a
// stretch of 32, of words r and r + 8 and of rows r, r + 8 of x; as the order of a dot product's terms is free, elements 0..3 of every
// lane make one warp product and 4..7 the next, which is how their fragments lie, with no exchange. The weight's pieces come by
// asynchronous copies into a ring of the thread's own, LOGIT_DEPTH steps of 128 elements ahead across the words' bounds; x lies in
// shared memory. The products of a step are added in f32 (the units cut what they add).
constexpr int LOGIT_DEPTH = 2, LOGIT_STEP = 128, LOGIT_THREADS = 512;
inline uint32_t few_x_pitch(uint64_t hidden) { return (uint32_t)((hidden + 127) / 128 * 128 + 32); }  // 64 bytes off a multiple of 128: no bank twice
template <typename T, int R>
__global__ void __launch_bounds__(LOGIT_THREADS) k_few_logits_16(const FewArgs a, uint32_t x_pitch) {
    static_assert(R == 8 || R == 16, "8 rows a product");
    extern __shared__ __align__(16) unsigned char ring[];  // [LOGIT_DEPTH][8][threads] 16 bytes, then x [R][x_pitch]
    __shared__ float2 by_warp[LOGIT_THREADS / 32][R];
    let_next();
    after_previous();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3;
    const T *x = static_cast<const T*>(a.x), *w = static_cast<const T*>(a.w);
    T* xs = reinterpret_cast<T*>(ring + LOGIT_DEPTH * 8 * LOGIT_THREADS * 16);
    const uint32_t tiles = (a.vocab + 15) / 16, steps = (a.hidden + LOGIT_STEP - 1) / LOGIT_STEP, stride = gridDim.x * (LOGIT_THREADS / 32);
    const uint32_t first = warp * gridDim.x + blockIdx.x;  // neighbours on neighbouring SMs
    uint32_t ft = first, fk = 0;  // what is fetched next: tile, step
    auto fetch = [&](uint32_t slot) {
        if (ft < tiles) {
            const T *w0 = w + (uint64_t)min(ft * 16 + r, a.vocab - 1) * a.hidden, *w1 = w + (uint64_t)min(ft * 16 + r + 8, a.vocab - 1) * a.hidden;
            const uint32_t to = smem_address(ring + (slot * 8 * LOGIT_THREADS + threadIdx.x) * 16), k = fk * LOGIT_STEP + 8 * q;
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (k + 32 * e < a.hidden) {
                    copy_async<16>(to + 2 * e * LOGIT_THREADS * 16, w0 + k + 32 * e);
                    copy_async<16>(to + (2 * e + 1) * LOGIT_THREADS * 16, w1 + k + 32 * e);
                }
        }
        copies_end();
        if (++fk == steps) {
            fk = 0;
            ft += stride;
        }
    };
#pragma unroll
    for (int e = 0; e < LOGIT_DEPTH; e++) fetch(e);
    for (uint32_t e = threadIdx.x; e < R * (x_pitch / 8); e += LOGIT_THREADS) {
        const uint32_t i = e / (x_pitch / 8), k = (e - i * (x_pitch / 8)) * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k < a.hidden && few_scored(a, i)) v = __ldg(reinterpret_cast<const uint4*>(x + (uint64_t)i * a.x_stride + k));
        *reinterpret_cast<uint4*>(xs + i * x_pitch + k) = v;
    }
    __syncthreads();
    float2 s[R / 8][2];
#pragma unroll
    for (int j = 0; j < R / 8; j++) s[j][0] = s[j][1] = make_float2(-INFINITY, 0.f);
    uint32_t slot = 0;
    for (uint32_t t = first; t < tiles; t += stride) {
        const uint32_t v0 = t * 16 + r, v1 = v0 + 8;
        float acc[R / 8][4] = {};
        for (uint32_t k0 = 0; k0 < a.hidden; k0 += LOGIT_STEP) {
            copies_but<LOGIT_DEPTH - 1>();
            const unsigned char* from = ring + (slot * 8 * LOGIT_THREADS + threadIdx.x) * 16;
            float c[R / 8][4] = {};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t k = k0 + 32 * e + 8 * q;
                uint4 p = make_uint4(0, 0, 0, 0), u = p;
                if (k < a.hidden) {
                    p = *reinterpret_cast<const uint4*>(from + 2 * e * LOGIT_THREADS * 16);
                    u = *reinterpret_cast<const uint4*>(from + (2 * e + 1) * LOGIT_THREADS * 16);
                }
#pragma unroll
                for (int j = 0; j < R / 8; j++) {
                    const uint4 y = *reinterpret_cast<const uint4*>(xs + (r + 8 * j) * x_pitch + k);
                    warp_product<T>(c[j], {p.x, u.x, p.y, u.y}, y.x, y.y);
                    warp_product<T>(c[j], {p.z, u.z, p.w, u.w}, y.z, y.w);
                }
            }
#pragma unroll
            for (int j = 0; j < R / 8; j++)
#pragma unroll
                for (int m = 0; m < 4; m++) acc[j][m] += c[j][m];
            fetch(slot);
            slot = slot + 1 == LOGIT_DEPTH ? 0 : slot + 1;
        }
        // this lane: words v0, v1 of rows 8 j + 2 q, + 1
#pragma unroll
        for (int j = 0; j < R / 8; j++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t v = h ? v1 : v0;
                if (v >= a.vocab) continue;
                if (a.finish) {
                    add_logit(s[j][0], acc[j][2 * h]);
                    add_logit(s[j][1], acc[j][2 * h + 1]);
                }
                *reinterpret_cast<float2*>(a.logits + (uint64_t)v * R + 8 * j + 2 * q) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
            }
    }
    copies_but<0>();
    if (!a.finish) return;
#pragma unroll
    for (int j = 0; j < R / 8; j++)
#pragma unroll
        for (int m = 0; m < 2; m++) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1)
                s[j][m] = join_stats(s[j][m], make_float2(__shfl_xor_sync(0xffffffffu, s[j][m].x, o), __shfl_xor_sync(0xffffffffu, s[j][m].y, o)));
            if (r == 0) by_warp[warp][8 * j + 2 * q + m] = s[j][m];
        }
    few_finish(a, by_warp);
}

// f32, and 16-bit rows off 16 bytes: a warp takes WORDS words, lanes along hidden; the rows of x are in shared memory as f32. A lane has 16
// bytes of a word at a time, by asynchronous copies as above (WIDE: f32 rows on 16 bytes), or one element.
template <typename T, int R, bool WIDE>
__global__ void __launch_bounds__(FEW_THREADS) k_few_logits(const FewArgs a) {
    static_assert(!WIDE || sizeof(T) == 4, "16-bit rows on 16 bytes go by warp products");
    constexpr int N = WIDE ? 16 / (int)sizeof(T) : 1, WORDS = 64 / R;
    constexpr int DEPTH = R == 4 ? 2 : R == 8 ? 3 : 4;
    extern __shared__ __align__(16) float xs[];  // [R][pitch], then (WIDE) the ring [DEPTH][WORDS][threads] 16 bytes
    __shared__ float2 by_warp[FEW_THREADS / 32][R];
    let_next();
    after_previous();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, pitch = (a.hidden + 32 * N - 1) / (32 * N) * (32 * N);
    const T *x = static_cast<const T*>(a.x), *w = static_cast<const T*>(a.w);
    const uint32_t tiles = (a.vocab + WORDS - 1) / WORDS, stride = gridDim.x * (FEW_THREADS / 32), first = blockIdx.x * (FEW_THREADS / 32) + warp;
    unsigned char* ring = reinterpret_cast<unsigned char*>(xs + R * pitch) + threadIdx.x * 16;
    uint32_t ft = first, fk = lane * N;  // what is fetched next: tile, element
    auto fetch = [&](uint32_t slot) {
        if (ft < tiles && fk < a.hidden) {
#pragma unroll
            for (int d = 0; d < WORDS; d++)
                copy_async<16>(smem_address(ring + (slot * WORDS + d) * FEW_THREADS * 16), w + (uint64_t)min(ft * WORDS + d, a.vocab - 1) * a.hidden + fk);
        }
        copies_end();
        fk += 32 * N;
        if (fk >= pitch) {
            fk = lane * N;
            ft += stride;
        }
    };
    if constexpr (WIDE) {
#pragma unroll
        for (int e = 0; e < DEPTH; e++) fetch(e);
    }
    for (uint32_t i = 0; i < R; i++) {
        const bool on = few_scored(a, i);
        for (uint32_t k = threadIdx.x; k < pitch; k += FEW_THREADS) xs[i * pitch + k] = on && k < a.hidden ? to_f32<T>(x[(uint64_t)i * a.x_stride + k]) : 0.f;
    }
    __syncthreads();
    // after the exchange below a lane has the logits of 64 / 32 = 2 (word, row) pairs
    float2 s[2] = {make_float2(-INFINITY, 0.f), make_float2(-INFINITY, 0.f)};
    uint32_t slot = 0;
    for (uint32_t t = first; t < tiles; t += stride) {
        float acc[64];  // [WORDS][R]
#pragma unroll
        for (int e = 0; e < 64; e++) acc[e] = 0.f;
        for (uint32_t k = lane * N; k < pitch; k += 32 * N) {
            Vec<T, N> v[WORDS];
            const bool in = k < a.hidden;
            if constexpr (WIDE) copies_but<DEPTH - 1>();
#pragma unroll
            for (int d = 0; d < WORDS; d++) {
                if (!in) continue;
                if constexpr (WIDE) v[d].q[0] = *reinterpret_cast<const uint4*>(ring + (slot * WORDS + d) * FEW_THREADS * 16);
                else v[d].load(w + (uint64_t)min(t * WORDS + d, a.vocab - 1) * a.hidden + k);
            }
#pragma unroll
            for (int i = 0; i < R; i++) {
                if (!in) continue;
                float y[N];
                if constexpr (N >= 4) {
#pragma unroll
                    for (int n = 0; n < N / 4; n++) *reinterpret_cast<float4*>(y + 4 * n) = *reinterpret_cast<const float4*>(xs + i * pitch + k + 4 * n);
                } else {
                    y[0] = xs[i * pitch + k];
                }
#pragma unroll
                for (int d = 0; d < WORDS; d++)
#pragma unroll
                    for (int n = 0; n < N; n++) acc[d * R + i] = fmaf(to_f32<T>(v[d].e[n]), y[n], acc[d * R + i]);
            }
            if constexpr (WIDE) {
                fetch(slot);
                slot = slot + 1 == DEPTH ? 0 : slot + 1;
            }
        }
        // 64 sums over 32 lanes: halves are exchanged, so that every lane ends with two of them
#pragma unroll
        for (int o = 16, n = 32; o; o >>= 1, n >>= 1) {
            const bool up = lane & o;
#pragma unroll
            for (int e = 0; e < 32; e++)
                if (e < n) {
                    const float give = up ? acc[e] : acc[e + n], keep = up ? acc[e + n] : acc[e];
                    acc[e] = keep + __shfl_xor_sync(0xffffffffu, give, o);
                }
        }
        // lane bits 16, 8, 4, 2, 1 chose the halves: its pair begins at 2 * lane (bit order kept)
        const uint32_t e0 = 2 * lane, word = t * WORDS + e0 / R, row = e0 % R;
        if (word < a.vocab) {
            if (a.finish) {
                add_logit(s[0], acc[0]);
                add_logit(s[1], acc[1]);
            }
            *reinterpret_cast<float2*>(a.logits + (uint64_t)word * R + row) = make_float2(acc[0], acc[1]);
        }
    }
    if constexpr (WIDE) copies_but<0>();
    if (!a.finish) return;
    // lanes with the same rows: those R / 2 apart
#pragma unroll
    for (int m = 0; m < 2; m++) {
#pragma unroll
        for (int o = R / 2; o < 32; o <<= 1)
            s[m] = join_stats(s[m], make_float2(__shfl_xor_sync(0xffffffffu, s[m].x, o), __shfl_xor_sync(0xffffffffu, s[m].y, o)));
        if (lane < R / 2) by_warp[warp][2 * lane + m] = s[m];
    }
    few_finish(a, by_warp);
}

// Four columns of a row: neighbours (WIDE: 4 elements as one access), or `across` apart.
template <typename T> struct alignas(4 * sizeof(T)) Four { T e[4]; };
template <typename T, bool WIDE>
__device__ __forceinline__ void load4(const T* row, uint32_t col0, uint32_t at, uint32_t across, uint32_t hidden, float (&v)[4]) {
    if constexpr (WIDE) {
        const Four<T> f = *reinterpret_cast<const Four<T>*>(row + col0 + 4 * at);
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = to_f32<T>(f.e[c]);
    } else {
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = col0 + at + c * across < hidden ? to_f32<T>(row[col0 + at + c * across]) : 0.f;
    }
}
template <typename T, bool WIDE>
__device__ __forceinline__ void store4(T* row, uint32_t col0, uint32_t at, uint32_t across, uint32_t hidden, const float (&v)[4]) {
    if constexpr (WIDE) {
        Four<T> f;
#pragma unroll
        for (int c = 0; c < 4; c++) f.e[c] = from_f32<T>(v[c]);
        *reinterpret_cast<Four<T>*>(row + col0 + 4 * at) = f;
    } else {
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (col0 + at + c * across < hidden) row[col0 + at + c * across] = from_f32<T>(v[c]);
    }
}

// Gradients. A thread has four columns of every row: x_i in registers, dX_i summed in registers; `along` threads share the words of a
// block where a row is shorter than the block (their sums are joined in order at the end).
template <typename T, typename G, int R, bool WIDE>
__global__ void __launch_bounds__(FEW_THREADS) k_few_grads(const FewArgs a, uint32_t across) {
    extern __shared__ __align__(16) float joined[];  // [along][R][4 * across], where along > 1
    __shared__ __align__(16) float g[FEW_WORDS][R];
    __shared__ float row_m[R], row_f[R], row_s[R];
    __shared__ uint32_t row_t[R];
    let_next();
    after_previous();
    const uint32_t along = FEW_THREADS / across, part = threadIdx.x / across, at = threadIdx.x - part * across;
    const uint32_t col0 = blockIdx.y * 4 * across;
    const T *x = static_cast<const T*>(a.x), *w = static_cast<const T*>(a.w);
    G* dw = static_cast<G*>(a.dw);
    auto column = [&](int c) { return col0 + (WIDE ? 4 * at + c : at + c * across); };
    if (threadIdx.x < R) {
        const uint32_t i = threadIdx.x;
        const bool on = few_scored(a, i);
        const float2 s = on ? a.stats[i] : make_float2(0.f, 1.f);
        row_m[i] = s.x;
        row_s[i] = s.y;
        row_f[i] = on ? (a.mask ? a.mask[i] : 1.f) / s.y : 0.f;
        row_t[i] = on ? (uint32_t)a.targets[i] : 0xffffffffu;
    }
    __syncthreads();
    float xr[R][4], sum[R][4];
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            xr[i][c] = row_t[i] != 0xffffffffu && column(c) < a.hidden ? to_f32<T>(x[(uint64_t)i * a.x_stride + column(c)]) : 0.f;
            sum[i][c] = 0.f;
        }
    const uint32_t begin = blockIdx.x * a.words, end = min(a.vocab, begin + a.words);
    // WIDE: a thread's pieces of the weight come by asynchronous copies into a ring of its own, DEPTH groups of AHEAD words ahead; only the
    // thread itself reads them, so no barrier is needed. `ahead` walks the words as the loops below do.
    constexpr int AHEAD = 4, DEPTH = 4;
    unsigned char* pipe = reinterpret_cast<unsigned char*>(joined) + threadIdx.x * sizeof(Four<T>);
    uint32_t slot = 0, ahead = begin + part;
    auto fetch = [&](uint32_t into) {
        const uint32_t stop = min(end, begin + ((ahead - begin) / FEW_WORDS + 1) * FEW_WORDS);  // of the stretch of FEW_WORDS that `ahead` is in
#pragma unroll
        for (int h = 0; h < AHEAD; h++)
            if (ahead + h * along < stop) copy_async<sizeof(Four<T>)>(smem_address(pipe + (into * AHEAD + h) * FEW_THREADS * sizeof(Four<T>)),
                                                                       w + (uint64_t)(ahead + h * along) * a.hidden + col0 + 4 * at);
        copies_end();
        ahead += AHEAD * along;
        if (ahead >= stop) ahead = stop + part;  // the stretch is done: the next begins with this thread's first word
    };
    if (WIDE && a.want_dx && column(0) < a.hidden)
        for (int e = 0; e < DEPTH; e++) fetch(e);
    for (uint32_t v0 = begin; v0 < end; v0 += FEW_WORDS) {
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < FEW_WORDS * R; e += FEW_THREADS) {
            const uint32_t v = v0 + e / R, i = e % R;
            float y = 0.f;
            if (v < end && row_t[i] != 0xffffffffu) {
                const float p = expf(a.logits[(uint64_t)v * R + i] - row_m[i]);
                y = (v == row_t[i] ? p - row_s[i] : p) * row_f[i];
            }
            g[e / R][i] = y;
        }
        __syncthreads();
        const uint32_t count = min((uint32_t)FEW_WORDS, end - v0);
        if (column(0) < a.hidden) {
            for (uint32_t d0 = part; d0 < count; d0 += AHEAD * along) {
                const uint32_t first = v0 + d0;
                float y[AHEAD][4], old[AHEAD][4];
                if constexpr (WIDE) {
                    if (a.want_dx) {  // the oldest of the thread's loads has come; the next takes its place once the words are done
                        copies_but<DEPTH - 1>();
#pragma unroll
                        for (int h = 0; h < AHEAD; h++) {
                            const Four<T> f = *reinterpret_cast<const Four<T>*>(pipe + (slot * AHEAD + h) * FEW_THREADS * sizeof(Four<T>));
#pragma unroll
                            for (int c = 0; c < 4; c++) y[h][c] = to_f32<T>(f.e[c]);
                        }
                    }
                } else if (a.want_dx) {
#pragma unroll
                    for (int h = 0; h < AHEAD; h++) load4<T, WIDE>(w + (uint64_t)(v0 + min(d0 + h * along, count - 1)) * a.hidden, col0, at, across, a.hidden, y[h]);
                }
                if (a.accumulate) {
#pragma unroll
                    for (int h = 0; h < AHEAD; h++) load4<G, WIDE>(dw + (uint64_t)(v0 + min(d0 + h * along, count - 1)) * a.hidden, col0, at, across, a.hidden, old[h]);
                }
#pragma unroll
                for (int h = 0; h < AHEAD; h++) {
                    const uint32_t d = d0 + h * along;
                    if (d >= count) break;
                    float out[4] = {};
#pragma unroll
                    for (int i = 0; i < R; i += 4) {
                        const float4 k4 = *reinterpret_cast<const float4*>(&g[d][i]);
                        const float k[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
                        for (int n = 0; n < 4; n++)
#pragma unroll
                            for (int c = 0; c < 4; c++) {
                                out[c] = fmaf(k[n], xr[i + n][c], out[c]);
                                if (a.want_dx) sum[i + n][c] = fmaf(k[n], y[h][c], sum[i + n][c]);
                            }
                    }
                    if (dw) {
#pragma unroll
                        for (int c = 0; c < 4; c++) out[c] = a.accumulate ? old[h][c] + out[c] * a.scale : out[c] * a.scale;
                        store4<G, WIDE>(dw + (uint64_t)(first + h * along) * a.hidden, col0, at, across, a.hidden, out);
                    }
                }
                if (WIDE && a.want_dx) {
                    fetch(slot);
                    slot = slot + 1 == DEPTH ? 0 : slot + 1;
                }
            }
        }
    }
    if constexpr (WIDE) copies_but<0>();
    if (!a.want_dx) return;
    float* to = a.dx_part + (uint64_t)blockIdx.x * R * a.hidden;
    if (along == 1) {
#pragma unroll
        for (int i = 0; i < R; i++) {
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (column(c) < a.hidden) to[(uint64_t)i * a.hidden + column(c)] = sum[i][c];
        }
        return;
    }
    __syncthreads();  // the ring and the sums share the memory
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) joined[(part * R + i) * 4 * across + (WIDE ? 4 * at + c : at + c * across)] = sum[i][c];
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < R * 4 * across; e += FEW_THREADS) {
        const uint32_t i = e / (4 * across), c = e - i * 4 * across;
        float t = 0.f;
        for (uint32_t p = 0; p < along; p++) t += joined[(p * R + i) * 4 * across + c];
        if (col0 + c < a.hidden) to[(uint64_t)i * a.hidden + col0 + c] = t;
    }
}

// Gradients of 16-bit operands on 16 bytes, by warp products. A block has 64 x across columns, a warp 64 of them; `along` = 4 / across
// warps share a stretch of 16 x along words. A stretch's piece of the weight (8 KiB) and its kept logits come by asynchronous copies
// GRAD_DEPTH stretches ahead; the block turns the logits into G, in two 16-bit parts (2^-16 of it is lost; one part would leave 2^-9,
// which so few rows do not average out: 0.0023 of the gradients of 16 rows instead of the 0.0017 that their own rounding is), of up to
// 8 rows the second in the place of rows 8 .. 15, of more as a product of its own (nothing, to 3 % at 128 columns) - and each warp multiplies
//   dX[i][h] += sum_v G[v][i] W[v][h]    A = G^T (words along K) and B = W, both through transposing loads
//   dW[v][h]  = sum_i G[v][i] x[i][h]    A = G as it lies, B = x in registers for good
// dW's columns are dealt to the product's so that a lane's 16 results of a word are neighbours, written as two pieces of 16 bytes.
constexpr int GRAD_DEPTH = 6, GRAD_THREADS = 128;
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrices_turned(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T, typename G, int R, int ACROSS_LOG>
__global__ void __launch_bounds__(GRAD_THREADS) k_few_grads_16(const FewArgs a) {
    extern __shared__ __align__(128) unsigned char raw16[];
    constexpr uint32_t across_log = ACROSS_LOG, across = 1u << ACROSS_LOG, along = 4 >> ACROSS_LOG, words = 16 * along;  // of a stretch
    constexpr uint32_t PIECE = 8192;
    constexpr bool SCALED = __is_same(T, __nv_bfloat16);  // bf16 has f32's range: the scale goes into G
    constexpr uint32_t l_bytes = words * R * 4;
    unsigned char* wp = raw16;                                                 // [GRAD_DEPTH][words][64 * across], 16-byte chunks turned by the word
    float* lp = reinterpret_cast<float*>(raw16 + GRAD_DEPTH * PIECE);          // [GRAD_DEPTH][words][R]
    T* gp = reinterpret_cast<T*>(raw16 + GRAD_DEPTH * (PIECE + l_bytes));      // [words][16], and of 16 rows the second parts behind
    __shared__ float row_m[16], row_f[16], row_s[16];
    __shared__ uint32_t row_t[16];
    let_next();
    after_previous();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, r = lane >> 2, q = lane & 3, mine = warp >> across_log, group = warp & (across - 1);
    const uint32_t col0 = blockIdx.y * 64 * across, col = col0 + group * 64;
    const T *x = static_cast<const T*>(a.x), *w = static_cast<const T*>(a.w);
    if (threadIdx.x < 16) {
        const uint32_t i = threadIdx.x;
        const bool on = i < R && few_scored(a, i);
        const float2 s = on ? a.stats[i] : make_float2(0.f, 1.f);
        row_m[i] = s.x;
        row_s[i] = s.y;
        row_f[i] = on ? (a.mask ? a.mask[i] : 1.f) / s.y * (SCALED ? a.scale : 1.f) : 0.f;
        row_t[i] = on ? (uint32_t)a.targets[i] : 0xffffffffu;
    }
    const uint32_t begin = blockIdx.x * a.words, end = min(a.vocab, begin + a.words), turns = (end - begin + words - 1) / words;
    auto fetch = [&](uint32_t turn) {
        if (turn < turns) {
            const uint32_t st = turn % GRAD_DEPTH, v0 = begin + turn * words;
            for (uint32_t e = threadIdx.x; e < PIECE / 16; e += GRAD_THREADS) {  // 16-byte chunk of a word
                const uint32_t d = e >> (3 + across_log), c = e & (8 * across - 1), at = col0 + 8 * c;
                const uint32_t to = smem_address(wp + st * PIECE + d * 128 * across + (c & ~7u) * 16 + (((c ^ d) & 7) << 4));
                if (v0 + d < end && at < a.hidden) copy_async<16>(to, w + (uint64_t)(v0 + d) * a.hidden + at);
                else asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to), "r"(0) : "memory");
            }
            for (uint32_t e = threadIdx.x; e < l_bytes / 16; e += GRAD_THREADS)
                if (v0 + e / (R / 4) < end) copy_async<16>(smem_address(reinterpret_cast<unsigned char*>(lp) + st * l_bytes + 16 * e), a.logits + (uint64_t)v0 * R + 4 * e);
        }
        copies_end();
    };
    for (int t = 0; t < GRAD_DEPTH - 1; t++) fetch(t);
    __syncthreads();
    // f16 holds 2^-24 .. 65504: G is scaled so that the largest weight times one goes to 2^13 .. 2^14
    float up = 1.f, down = 1.f;
    if constexpr (__is_same(T, __half)) {
        float top = 0.f;
        for (int i = 0; i < R; i++) top = fmaxf(top, row_t[i] != 0xffffffffu ? (a.mask ? fabsf(a.mask[i]) : 1.f) : 0.f);
        const int e = top > 0.f && isfinite(top) ? min(max(13 - ilogbf(top), -100), 100) : 0;
        up = exp2f((float)e);
        down = exp2f((float)-e);
    }
    // x for dW: column n of product j is column 16 (n / 2) + 2 j + n % 2 of the warp's 64
    uint32_t xb[8][2];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t h = col + 16 * (r >> 1) + 2 * j + (r & 1);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            T v[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint32_t i = (R == 8 ? 0 : 8 * k) + 2 * q + e;
                v[e] = h < a.hidden && row_t[i] != 0xffffffffu ? x[(uint64_t)i * a.x_stride + h] : from_f32<T>(0.f);
            }
            xb[j][k] = (uint32_t)*reinterpret_cast<uint16_t*>(&v[0]) | (uint32_t)*reinterpret_cast<uint16_t*>(&v[1]) << 16;
        }
    }
    float dx[8][4];
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
        for (int m = 0; m < 4; m++) dx[j][m] = 0.f;
    G* dw = static_cast<G*>(a.dw);
    const float out_scale = SCALED ? 1.f : a.scale * down, dx_scale = SCALED ? 1.f : a.scale * down;
    for (uint32_t turn = 0; turn < turns; turn++) {
        const uint32_t st = turn % GRAD_DEPTH, v0 = begin + turn * words;
        copies_but<GRAD_DEPTH - 2>();
        __syncthreads();  // this stretch is here for everyone, and everyone is done with the one before
        fetch(turn + GRAD_DEPTH - 1);
        for (uint32_t e = threadIdx.x; e < words * R; e += GRAD_THREADS) {
            const uint32_t d = e / R, i = e % R, v = v0 + d;
            float y = 0.f;
            if (v < end && row_t[i] != 0xffffffffu) {
                float p;  // 2^-22 is ample for 16 bits, twice
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"((lp[st * words * R + e] - row_m[i]) * 1.4426950408889634f));
                y = (v == row_t[i] ? p - row_s[i] : p) * row_f[i] * up;
            }
            const T hi = from_f32<T>(y), lo = from_f32<T>(isfinite(y) ? y - to_f32<T>(hi) : 0.f);
            gp[d * 16 + i] = hi;
            gp[R == 8 ? d * 16 + 8 + i : (words + d) * 16 + i] = lo;
        }
        __syncthreads();
        if (col >= a.hidden) continue;
        constexpr int PARTS = R / 8;
        uint32_t gt[PARTS][4], gn[PARTS][4];  // G^T and G of the warp's 16 words
#pragma unroll
        for (int p = 0; p < PARTS; p++) {
            const T* from = gp + (p * words + mine * 16) * 16;
            load_matrices_turned(gt[p], smem_address(from + ((lane >> 4) * 8 + (lane & 7)) * 16 + ((lane >> 3) & 1) * 8));
            load_matrices(gn[p], smem_address(from + (((lane >> 3) & 1) * 8 + (lane & 7)) * 16 + (lane >> 4) * 8));
        }
        if (a.want_dx) {
            const unsigned char* piece = wp + st * PIECE;
            const uint32_t d = mine * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);  // the word this lane points at
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                uint32_t b[4];
                const uint32_t c = j + (lane >> 4);
                load_matrices_turned(b, smem_address(piece + d * 128 * across + group * 128 + (((c ^ d) & 7) << 4)));
#pragma unroll
                for (int p = PARTS - 1; p >= 0; p--) {
                    warp_product<T>(dx[j], gt[p], b[0], b[1]);
                    warp_product<T>(dx[j + 1], gt[p], b[2], b[3]);
                }
            }
        }
        if (dw) {
            float out[8][4];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                out[j][0] = out[j][1] = out[j][2] = out[j][3] = 0.f;
#pragma unroll
                for (int p = PARTS - 1; p >= 0; p--) warp_product<T>(out[j], gn[p], xb[j][0], xb[j][1]);
            }
            const uint32_t h = col + 16 * q;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const uint32_t v = v0 + mine * 16 + r + 8 * k;
                if (v >= end) continue;
                G* to = dw + (uint64_t)v * a.hidden + h;
#pragma unroll
                for (int e = 0; e < 2; e++) {  // 8 columns: whole 16-byte pieces, as rows are
                    if (h + 8 * e >= a.hidden) break;
                    float y[8];
#pragma unroll
                    for (int c = 0; c < 8; c++) y[c] = SCALED ? out[4 * e + c / 2][2 * k + (c & 1)] : out[4 * e + c / 2][2 * k + (c & 1)] * out_scale;
                    Vec<G, 8> o;
                    if (a.accumulate) {
                        o.load_coherent(to + 8 * e);
#pragma unroll
                        for (int c = 0; c < 8; c++) y[c] += to_f32<G>(o.e[c]);
                    }
                    o.q[0] = make_uint4(pack2<G>(y[0], y[1]), pack2<G>(y[2], y[3]), pack2<G>(y[4], y[5]), pack2<G>(y[6], y[7]));
                    o.store(to + 8 * e);
                }
            }
        }
    }
    copies_but<0>();
    if (!a.want_dx) return;
    float* to = a.dx_part + (uint64_t)blockIdx.x * R * a.hidden;
    float* sums = reinterpret_cast<float*>(raw16);  // [along][16][64 * across]
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
        for (int m = 0; m < 4; m++) sums[((mine * 16) + r + 8 * (m >> 1)) * 64 * across + group * 64 + 8 * j + 2 * q + (m & 1)] = dx[j][m] * dx_scale;
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < R * 64 * across; e += GRAD_THREADS) {
        const uint32_t i = e / (64 * across), c = e - i * 64 * across;
        float t = 0.f;
        for (uint32_t p = 0; p < along; p++) {
            t += sums[(p * 16 + i) * 64 * across + c];
            if (R == 8) t += sums[(p * 16 + 8 + i) * 64 * across + c];
        }
        if (col0 + c < a.hidden) to[(uint64_t)i * a.hidden + col0 + c] = t;
    }
}

// d_hidden: the blocks' sums in order, eight warps a part each, joined in order. A block has one row and 32 columns.
template <typename T, int R>
__global__ void __launch_bounds__(256) k_few_d_hidden(const FewArgs a, uint32_t parts, float scale) {
    __shared__ float share[8][32];
    let_next();
    after_previous();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31, i = blockIdx.y, col = blockIdx.x * 32 + lane;
    const bool on = few_scored(a, i);
    float t = 0.f;
    if (on && col < a.hidden) {
        const uint32_t each = (parts + 7) / 8, p1 = min(parts, (warp + 1) * each);
#pragma unroll 8
        for (uint32_t p = warp * each; p < p1; p++) t += a.dx_part[((uint64_t)p * R + i) * a.hidden + col];
    }
    share[warp][lane] = t;
    __syncthreads();
    if (warp || col >= a.hidden) return;
#pragma unroll
    for (int w = 1; w < 8; w++) t += share[w][lane];
    static_cast<T*>(a.dx)[(uint64_t)i * a.dx_stride + col] = from_f32<T>(on ? t * scale : 0.f);
}

// ---- the launches of one call
inline uint32_t few_across(uint64_t hidden) {  // threads of a block along a row
    uint32_t n = 8;
    while (n < (uint32_t)FEW_THREADS && (uint64_t)n * 4 < hidden) n *= 2;
    return n;
}
// Blocks along the vocabulary of the gradients' kernels, over all column tiles one round of what the SMs hold: k_few_grads one block an SM
// (two where eight rows or fewer leave the registers), 32 words a block at least; k_few_grads_16 four, two stretches at least.
inline uint32_t few_parts(uint64_t hidden, uint64_t vocab, int sms, int rows) {
    const uint32_t across = few_across(hidden), columns = (uint32_t)((hidden + 4 * across - 1) / (4 * across));
    const uint64_t most = (vocab + 31) / 32, want = std::max<uint64_t>(1, (uint64_t)sms * (rows > 8 ? 1 : 2) / columns);
    return (uint32_t)std::min(want, most);
}
inline uint32_t few_across_16(uint64_t hidden) { return hidden > 128 ? 4 : hidden > 64 ? 2 : 1; }
inline uint32_t few_parts_16(uint64_t hidden, uint64_t vocab, int sms) {
    const uint32_t across = few_across_16(hidden), columns = (uint32_t)((hidden + 64 * across - 1) / (64 * across)), words = 64 / across;
    const uint64_t most = (vocab + 2 * words - 1) / (2 * words), want = std::max<uint64_t>(1, (uint64_t)sms * 4 / columns);
    return (uint32_t)std::min(want, most);
}
constexpr int FEW_LOGIT_BLOCKS = 4;  // blocks of k_few_logits* an SM
constexpr int FEW_GRAD_BYTES = FEW_THREADS * 4 * FEW_ROWS * 4;  // k_few_grads: the ring of copies, or the joined sums
constexpr size_t FEW_SHARED = 227 << 10;   // what a block can have
// The rows a kernel is made for that serves `rows`.
inline int few_kernel_rows(uint64_t rows, size_t size, bool wide) { return rows <= 4 && !(size == 2 && wide) ? 4 : rows <= 8 ? 8 : 16; }
// Shared memory of the logits' kernel: the rows of x and the ring of copies.
inline size_t few_logit_bytes(int r, uint64_t hidden, size_t size, bool wide) {
    if (size == 2 && wide) return LOGIT_DEPTH * 8 * LOGIT_THREADS * 16 + (size_t)r * few_x_pitch(hidden) * 2;
    const uint64_t n = wide ? 16 / size : 1, pitch = (hidden + 32 * n - 1) / (32 * n) * (32 * n);
    return (size_t)r * pitch * 4 + (wide ? (size_t)(r == 4 ? 2 : r == 8 ? 3 : 4) * (64 / r) * FEW_THREADS * 16 : 0);
}
// More than 8 rows of 16-bit values that do not lie on 16 bytes go this way only over a small weight: read by elements, 16 rows of
// 345 x 20000 take 42 us for the losses and 91 with gradients, where the tiles take 24 and 67 (97 x 100000: 52 and 116, 38 and 123;
// 97 x 2000: 13 and 27, 14 and 33).
inline bool few_fits(uint64_t rows, uint64_t hidden, uint64_t vocab, size_t size, bool wide) {
    if (size == 2 && !wide && rows > 8 && hidden * vocab > (1u << 20)) return false;
    return rows <= (uint64_t)FEW_ROWS && few_logit_bytes(few_kernel_rows(rows, size, wide), hidden, size, wide) + 8192 <= FEW_SHARED;
}
// Every batch of up to `rows` rows goes this way, wherever its rows lie; *most: the rows of the largest kernel among them.
inline bool few_always(uint64_t rows, uint64_t hidden, uint64_t vocab, size_t size, int* most) {
    *most = 0;
    if (rows > (uint64_t)FEW_ROWS) return false;
    for (uint64_t r = 0; r <= rows; r++)
        for (const bool wide : {false, true}) {
            if (wide && hidden * size % 16 != 0) continue;
            if (!few_fits(r, hidden, vocab, size, wide)) return false;
            *most = std::max(*most, few_kernel_rows(r, size, wide));
        }
    return true;
}
template <typename T, int R>
int32_t few_logits(const FewArgs& a, bool wide, int sms, cudaStream_t s) {
    const size_t shared = few_logit_bytes(R, a.hidden, sizeof(T), wide);
    const uint32_t fit = std::max<uint32_t>(1, std::min<uint32_t>(FEW_LOGIT_BLOCKS, (uint32_t)((220 << 10) / shared)));
    auto blocks = [&](uint32_t words) { return std::min<uint32_t>(((a.vocab + words - 1) / words + 7) / 8, sms * fit); };
    if constexpr (sizeof(T) == 2 && R >= 8) {
        if (wide) {
            OXZ_CUDA(launch_after(false, k_few_logits_16<T, R>, std::min<uint32_t>((a.vocab + 15) / 16, sms), LOGIT_THREADS, shared, s, a, few_x_pitch(a.hidden)));
            return OXZ_OK;
        }
    }
    auto k = k_few_logits<T, R, false>;
    if constexpr (sizeof(T) == 4) {  // 16-bit rows on 16 bytes have gone the other way
        if (wide) k = k_few_logits<T, R, true>;
    }
    OXZ_CUDA(launch_after(false, k, blocks(64 / R), FEW_THREADS, shared, s, a));
    return OXZ_OK;
}

// wide: the rows of x and of the weight lie on 16 bytes. out_wide: four elements of a row of the weight, of x and of d_weight are one access.
template <typename T, typename G, int R>
int32_t few_run_rows(FewArgs a, bool wide, bool out_wide, bool grads, int sms, cudaStream_t s) {
    OXZ_TRY((few_logits<T, R>(a, wide, sms, s)));
    if (!grads) return OXZ_OK;
    uint32_t parts = 0;
    bool scaled = false;  // the partial sums carry the scale already
    if constexpr (sizeof(T) == 2 && sizeof(G) == 2 && R >= 8) {  // (an f32 d_weight wants G in f32)
        if (wide) {
            const uint32_t across = few_across_16(a.hidden), columns = (a.hidden + 64 * across - 1) / (64 * across), words = 64 / across;
            parts = few_parts_16(a.hidden, a.vocab, sms);
            a.words = ((a.vocab + parts - 1) / parts + words - 1) / words * words;
            parts = (a.vocab + a.words - 1) / a.words;
            const size_t shared = (size_t)GRAD_DEPTH * (8192 + words * R * 4) + words * 16 * 2 * (R / 8);
            auto k = across == 4 ? k_few_grads_16<T, G, R, 2> : across == 2 ? k_few_grads_16<T, G, R, 1> : k_few_grads_16<T, G, R, 0>;
            OXZ_CUDA(launch_after(true, k, dim3(parts, columns), GRAD_THREADS, shared, s, a));
            scaled = true;
        }
    }
    if (!scaled) {
        const uint32_t across = few_across(a.hidden), columns = (a.hidden + 4 * across - 1) / (4 * across);
        parts = few_parts(a.hidden, a.vocab, sms, R);
        a.words = (a.vocab + parts - 1) / parts;
        parts = (a.vocab + a.words - 1) / a.words;
        auto k = out_wide ? k_few_grads<T, G, R, true> : k_few_grads<T, G, R, false>;
        OXZ_CUDA(launch_after(true, k, dim3(parts, columns), FEW_THREADS, FEW_GRAD_BYTES, s, a, across));
    }
    if (a.want_dx && a.rows)
        OXZ_CUDA(launch_after(true, k_few_d_hidden<T, R>, dim3((a.hidden + 31) / 32, a.rows), 256, 0, s, a, parts, scaled ? 1.f : a.scale));
    return OXZ_OK;
}
template <typename T, typename G>
int32_t few_run(const FewArgs& a, bool wide, bool out_wide, bool grads, int sms, cudaStream_t s) {
    const int r = few_kernel_rows(a.rows, sizeof(T), wide);
    if (r == 4) return few_run_rows<T, G, 4>(a, wide, out_wide, grads, sms, s);
    if (r == 8) return few_run_rows<T, G, 8>(a, wide, out_wide, grads, sms, s);
    return few_run_rows<T, G, 16>(a, wide, out_wide, grads, sms, s);
}
// The shared memory that the kernels may need, granted once.
template <typename T, typename G, int R>
int32_t few_prepare_rows() {
    if constexpr (sizeof(T) == 4) OXZ_CUDA(cudaFuncSetAttribute(k_few_logits<T, R, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FEW_SHARED - 4096));
    OXZ_CUDA(cudaFuncSetAttribute(k_few_logits<T, R, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FEW_SHARED - 4096));
    OXZ_CUDA(cudaFuncSetAttribute(k_few_grads<T, G, R, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_GRAD_BYTES));
    OXZ_CUDA(cudaFuncSetAttribute(k_few_grads<T, G, R, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_GRAD_BYTES));
    if constexpr (sizeof(T) == 2 && R >= 8) OXZ_CUDA(cudaFuncSetAttribute(k_few_logits_16<T, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)FEW_SHARED - 4096));
    if constexpr (sizeof(T) == 2 && sizeof(G) == 2 && R >= 8) {
        OXZ_CUDA(cudaFuncSetAttribute(k_few_grads_16<T, G, R, 0>, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 << 10));
        OXZ_CUDA(cudaFuncSetAttribute(k_few_grads_16<T, G, R, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 << 10));
        OXZ_CUDA(cudaFuncSetAttribute(k_few_grads_16<T, G, R, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, 96 << 10));
    }
    return OXZ_OK;
}
template <typename T, typename G>
int32_t few_prepare() {
    OXZ_TRY((few_prepare_rows<T, G, 4>()));
    OXZ_TRY((few_prepare_rows<T, G, 8>()));
    return few_prepare_rows<T, G, 16>();
}

}  // namespace
}  // namespace oxz
