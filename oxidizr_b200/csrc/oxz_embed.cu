// The token embedding (oxz_embed_*): a scaled row lookup, and its gradient by sorted tokens.
//
//   out[i] = c * T[id_i]            dT[v] = c * sum_{i : id_i = v} dY_i   (+ dT[v])
//
// Both are bound by memory: the lookup reads and writes n rows; the gradient reads n rows and writes either the whole table
// (overwriting) or the rows that have tokens, read and written (accumulating). The gradient adds no atomics: the tokens are
// sorted (stable, so equal tokens keep their order), every sum runs in f32 in that order, and equal inputs give equal bits.
#include <algorithm>
#include <cmath>

#include <cooperative_groups.h>

#include "oxz_elem.cuh"
#include "oxz_internal.h"

namespace cg = cooperative_groups;

struct oxz_embed {
    oxz_embed_desc d{};
    bool allocated = false;
    uint64_t bytes = 0;
    unsigned long long* sorted[2] = {nullptr, nullptr};  // token << 32 | position, max_tokens each
    float* carry = nullptr;                              // [chunks][2][hidden]: partial sums of the tokens that cross chunks
    uint32_t* touched = nullptr;                         // a bit for every row of the table: it has a token. All 0 between calls
    bool clean = false;                                  // ... unless a call broke off, and clearing them failed as well
    int sms = 0;
    oxz::StreamOrder order;
};

namespace oxz {
namespace {

constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32, SORT_CLUSTER = 8;
constexpr int DIGIT_BITS = 9, BINS = 1 << DIGIT_BITS;
constexpr uint32_t CHUNK = 16;  // sorted tokens a warp sums on its own
constexpr uint32_t DIRECT = 1024;  // tokens that are summed without being sorted: see k_embed_direct
constexpr uint32_t RANKED = 8192;  // tokens that are sorted by counting: see k_embed_rank

// ---- lookup: a warp takes a piece of 32 x 4 vectors of one row
template <typename T, int N>
__global__ void __launch_bounds__(256) k_embed_lookup(const int64_t* __restrict__ ids, uint64_t n, const T* __restrict__ table,
                                                      T* __restrict__ out, uint64_t out_stride, uint32_t hidden, uint64_t vocab,
                                                      float scale, uint32_t pieces) {
    for (uint64_t unit = (uint64_t)blockIdx.x * 8 + threadIdx.x / 32; unit < n * pieces; unit += (uint64_t)gridDim.x * 8) {
        const uint64_t row = unit / pieces;
        const uint32_t first = (uint32_t)(unit - row * pieces) * 32 * 4 * N + (threadIdx.x & 31) * N;
        const int64_t id = ids[row];
        const bool known = (uint64_t)id < vocab;
        const T* src = table + (known ? (uint64_t)id * hidden : 0);
        T* dst = out + row * out_stride;
        Vec<T, N> v[4];
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (known && first + k * 32 * N < hidden) v[k].load(src + first + k * 32 * N);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (first + k * 32 * N >= hidden) break;
#pragma unroll
            for (int j = 0; j < N; j++) v[k].e[j] = from_f32<T>(known ? to_f32<T>(v[k].e[j]) * scale : 0.f);
            v[k].store(dst + first + k * 32 * N);
        }
    }
}

// ---- gradient, first launch: the tokens sorted, by one cluster of blocks.
//
// The sort is a least-significant-digit radix sort by digits of at most 9 bits. A block owns a contiguous run of the items, a
// warp a contiguous run of the block's, and walks it 32 at a time: __match_any_sync ranks equal digits within the 32, a
// histogram of the warp's own counts the ones before. Bases come from the blocks' histograms, read through distributed shared
// memory, so that a pass is: count, cluster barrier, place, cluster barrier. Ids outside the table get the key `vocab`, sort
// behind every token and are not summed.
struct SortShared {
    uint32_t mine[SORT_WARPS][BINS];  // per warp: items of each digit seen (first walk), then the next place (second walk)
    uint32_t block[BINS];             // the block's histogram, read by the other blocks
    uint32_t scan[SORT_WARPS];
};

__device__ void sort_tokens(cg::cluster_group& cl, SortShared& sh, const int64_t* __restrict__ ids, uint32_t n, uint32_t vocab,
                            int passes, int bits, unsigned long long* a, unsigned long long* b) {
    const uint32_t rank = cl.block_rank(), blocks = cl.num_blocks();
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const uint32_t bins = 1u << bits;
    // runs are multiples of 32 items so that only the last warp with items meets a part of 32
    const uint32_t per_warp = (((n + blocks * SORT_WARPS - 1) / (blocks * SORT_WARPS)) + 31) & ~31u;
    const uint64_t begin = (uint64_t)(rank * SORT_WARPS + warp) * per_warp;
    const uint32_t lo = (uint32_t)min(begin, (uint64_t)n), hi = (uint32_t)min(begin + per_warp, (uint64_t)n);
    unsigned long long *src = a, *dst = b;
    for (int pass = 0; pass < passes; pass++) {
        const int shift = pass * bits;
        auto item = [&](uint32_t i) -> unsigned long long {
            if (pass == 0) {
                const int64_t id = ids[i];
                return (unsigned long long)((uint64_t)id < vocab ? (uint32_t)id : vocab) << 32 | i;
            }
            return src[i];
        };
        for (uint32_t i = threadIdx.x; i < SORT_WARPS * bins; i += SORT_THREADS) sh.mine[i / bins][i % bins] = 0;
        __syncthreads();
        for (uint32_t i0 = lo; i0 < hi; i0 += 32) {
            const bool have = i0 + lane < hi;
            const uint32_t digit = have ? (uint32_t)(item(i0 + lane) >> (32 + shift)) & (bins - 1) : bins;
            const uint32_t same = __match_any_sync(0xffffffffu, digit);
            if (have && lane == (uint32_t)(__ffs(same) - 1)) sh.mine[warp][digit] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
        for (uint32_t d = threadIdx.x; d < bins; d += SORT_THREADS) {
            uint32_t sum = 0;
            for (int w = 0; w < SORT_WARPS; w++) sum += sh.mine[w][d];
            sh.block[d] = sum;
        }
        cl.sync();
        // thread d: the items of its digit in all blocks, and in the blocks before this one
        uint32_t total = 0, before = 0;
        if (threadIdx.x < bins) {
            for (uint32_t r = 0; r < blocks; r++) {
                const uint32_t c = cl.map_shared_rank(sh.block, r)[threadIdx.x];
                total += c;
                before += r < rank ? c : 0;
            }
        }
        // exclusive scan of the totals over the digits
        uint32_t inc = total;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= (uint32_t)o) inc += up;
        }
        if (lane == 31) sh.scan[warp] = inc;
        __syncthreads();
        if (warp == 0) {
            uint32_t w = sh.scan[lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xffffffffu, w, o);
                if (lane >= (uint32_t)o) w += up;
            }
            sh.scan[lane] = w;
        }
        __syncthreads();
        if (threadIdx.x < bins) {
            uint32_t place = inc - total + (warp ? sh.scan[warp - 1] : 0) + before;
            for (int w = 0; w < SORT_WARPS; w++) {
                const uint32_t c = sh.mine[w][threadIdx.x];
                sh.mine[w][threadIdx.x] = place;
                place += c;
            }
        }
        __syncthreads();
        for (uint32_t i0 = lo; i0 < hi; i0 += 32) {
            const bool have = i0 + lane < hi;
            const unsigned long long it = have ? item(i0 + lane) : 0;
            const uint32_t digit = have ? (uint32_t)(it >> (32 + shift)) & (bins - 1) : bins;
            const uint32_t same = __match_any_sync(0xffffffffu, digit);
            uint32_t place = 0;
            if (have) place = sh.mine[warp][digit] + __popc(same & ((1u << lane) - 1));
            __syncwarp();
            if (have && lane == (uint32_t)(__ffs(same) - 1)) sh.mine[warp][digit] += __popc(same);
            __syncwarp();
            if (have) dst[place] = it;
        }
        cl.sync();  // the items are in place for every block, and nobody reads this pass's histograms any more
        unsigned long long* t = src;
        src = dst;
        dst = t;
    }
}

// A table that is overwritten is filled with zeros where no token is: the first launch marks the rows that have one.
__device__ __forceinline__ void mark(uint32_t* touched, uint32_t key, uint32_t vocab) {
    if (touched && key < vocab) atomicOr(&touched[key >> 5], 1u << (key & 31));
}

__global__ void __launch_bounds__(SORT_THREADS) k_embed_sort(const int64_t* __restrict__ ids, uint32_t n, uint32_t vocab, int passes,
                                                             int bits, unsigned long long* a, unsigned long long* b, uint32_t* touched) {
    extern __shared__ __align__(16) unsigned char raw[];
    let_next();
    cg::cluster_group cl = cg::this_cluster();
    sort_tokens(cl, *reinterpret_cast<SortShared*>(raw), ids, n, vocab, passes, bits, a, b);
    for (uint32_t i = blockIdx.x * SORT_THREADS + threadIdx.x; i < n; i += gridDim.x * SORT_THREADS) {
        const int64_t id = ids[i];
        mark(touched, (uint64_t)id < vocab ? (uint32_t)id : vocab, vocab);
    }
}

// ---- gradient, first launch, up to RANKED tokens: a token's place is the count of tokens with a smaller id, and of equal ones before it.
// The tokens are dealt evenly to one block an SM; PARTS threads a token count over a share of all tokens in shared memory each, 32 while
// a block has no more than 32 tokens. 8192 tokens take 7 us, where the radix sort's barriers take 16; see the sums for whole calls.
template <int PARTS>
__global__ void __launch_bounds__(SORT_THREADS) k_embed_rank(const int64_t* __restrict__ ids, uint32_t n, uint32_t vocab, uint32_t tokens,
                                                             unsigned long long* sorted, uint32_t* touched) {
    __shared__ __align__(16) uint32_t key[RANKED];
    let_next();
    const uint32_t padded = (n + 4 * PARTS - 1) / (4 * PARTS) * (4 * PARTS);
    for (uint32_t i = threadIdx.x; i < padded; i += blockDim.x) {
        const int64_t id = i < n ? ids[i] : -1;
        key[i] = i < n ? ((uint64_t)id < vocab ? (uint32_t)id : vocab) : 0xffffffffu;
    }
    __syncthreads();
    const uint32_t own = threadIdx.x / PARTS, part = threadIdx.x % PARTS;
    const bool here = own < tokens && blockIdx.x * tokens + own < n;
    const uint32_t i = here ? blockIdx.x * tokens + own : 0, mine = key[i];
    uint32_t count = 0;
    // in front of the token equal ids count too; its own four are looked at one by one
    auto four = [&](uint32_t j) { return *reinterpret_cast<const uint4*>(key + j); };
    const uint32_t its = i & ~3u;
    uint32_t j = part * 4;
#pragma unroll 4
    for (; j < its; j += 4 * PARTS) {
        const uint4 k = four(j);
        count += (k.x <= mine) + (k.y <= mine) + (k.z <= mine) + (k.w <= mine);
    }
    if (j == its && here) {
        for (uint32_t e = j; e < j + 4; e++) count += key[e] < mine + (e < i);
        j += 4 * PARTS;
    }
#pragma unroll 4
    for (; j < padded; j += 4 * PARTS) {
        const uint4 k = four(j);
        count += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
    }
#pragma unroll
    for (int o = PARTS / 2; o; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
    if (part == 0 && here) {
        sorted[count] = (unsigned long long)mine << 32 | i;
        mark(touched, mine, vocab);
    }
}
// Zeros over one row, by a warp
__device__ __forceinline__ void fill_row(unsigned char* row, uint64_t bytes) {
    const uint32_t lane = threadIdx.x & 31;
    unsigned char* lo = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(row) + 31) & ~(uintptr_t)31);
    const uint64_t head = min((uint64_t)(lo - row), bytes), pieces = (bytes - head) / 32, tail = bytes - head - pieces * 32;
    const uint32_t zero[8] = {};
    for (uint64_t i = lane; i < pieces; i += 32) store32(lo + 32 * i, zero);
    if (lane < head) row[lane] = 0;
    if (lane < tail) lo[pieces * 32 + lane] = 0;
}

__device__ __forceinline__ uint32_t key_of(unsigned long long it) { return (uint32_t)(it >> 32); }

// v: what the row holds, where it is added to
template <typename G, int N>
__device__ __forceinline__ void write_row(G* dst, Vec<G, N>& v, const float (&sum)[N], float scale, bool accumulate) {
#pragma unroll
    for (int j = 0; j < N; j++) v.e[j] = from_f32<G>(accumulate ? to_f32<G>(v.e[j]) + sum[j] * scale : sum[j] * scale);
    v.store(dst);
}
template <typename G, int N>
__device__ __forceinline__ void write_row(G* dst, const float (&sum)[N], float scale, bool accumulate) {
    Vec<G, N> v;
    if (accumulate) v.load_coherent(dst);
    write_row<G, N>(dst, v, sum, scale, accumulate);
}

// ---- gradient, second launch: a warp sums one chunk of CHUNK sorted tokens for 32 x N columns. Tokens that lie inside the
// chunk are written; the sums of a token that goes on from the chunk before or into the chunk after go to the carries:
// carry[chunk][0] for the token the chunk begins with, carry[chunk][1] for one that begins in the chunk and leaves it.
// Blocks from `summing` on write zeros to the rows that have no token: the sums wait on their loads, the zeros take the memory meanwhile
// (a fill of all rows beside the sort, and the sums after it, took 9 us more: 8192 x 2048 bf16, 128256 rows, 117 us now). Where rows are
// added to (ADD), what they hold is asked for along with the rows that are summed: 39 us instead of 46 (4974 x 448: 20 instead of 25).
template <typename T, typename G, int N, bool ADD>
__global__ void __launch_bounds__(256) k_embed_sums(const unsigned long long* __restrict__ sorted, uint32_t n, uint32_t vocab,
                                                    const T* __restrict__ d_out, uint64_t stride, uint32_t hidden, G* d_table,
                                                    float* __restrict__ carry, float scale, uint32_t slices, uint32_t summing,
                                                    const uint32_t* __restrict__ touched) {
    let_next();
    after_previous();
    if (blockIdx.x >= summing) {
        // a warp takes 8 rows, and asks for the next ones' bits before it writes
        const uint64_t row_bytes = (uint64_t)hidden * sizeof(G), warps = (uint64_t)(gridDim.x - summing) * 8, eights = ((uint64_t)vocab + 7) / 8;
        const unsigned char* bits_of = reinterpret_cast<const unsigned char*>(touched);
        uint64_t u = (uint64_t)(blockIdx.x - summing) * 8 + threadIdx.x / 32;
        uint32_t next = u < eights ? bits_of[u] : 0;
        for (; u < eights; u += warps) {
            const uint32_t bits = next;
            if (u + warps < eights) next = bits_of[u + warps];
            const uint32_t rows = (uint32_t)min((uint64_t)8, vocab - u * 8);
            for (uint32_t r = 0; r < rows; r++)
                if (!(bits >> r & 1)) fill_row(reinterpret_cast<unsigned char*>(d_table) + (u * 8 + r) * row_bytes, row_bytes);
        }
        return;
    }
    const uint64_t chunks = (n + CHUNK - 1) / CHUNK;
    const uint32_t lane = threadIdx.x & 31;
    for (uint64_t unit = (uint64_t)blockIdx.x * 8 + threadIdx.x / 32; unit < chunks * slices; unit += (uint64_t)summing * 8) {
        const uint32_t chunk = (uint32_t)(unit / slices);
        const uint64_t c0 = (uint64_t)chunk * CHUNK;
        const uint32_t col = (uint32_t)(unit - (uint64_t)chunk * slices) * 32 * N + lane * N;
        const uint32_t count = (uint32_t)min((uint64_t)CHUNK, n - c0);
        // lane k holds item k; lane CHUNK the item after the chunk
        unsigned long long it = (unsigned long long)vocab << 32;
        if (lane < count || (lane == count && c0 + count < n)) it = sorted[c0 + lane];
        const uint32_t first_key = __shfl_sync(0xffffffffu, key_of(it), 0);
        const bool from_left = c0 > 0 && key_of(sorted[c0 - 1]) == first_key;
        const bool live = col < hidden;
        float sum[N];
#pragma unroll
        for (int j = 0; j < N; j++) sum[j] = 0.f;
        uint32_t begin = 0;  // where the current token's run begins in the chunk
        constexpr int AHEAD = ADD ? 4 : 8;
        for (uint32_t k0 = 0; k0 < count; k0 += AHEAD) {
            Vec<T, N> v[AHEAD];
            Vec<G, N> old[ADD ? AHEAD : 1];
#pragma unroll
            for (int a = 0; a < AHEAD; a++) {
                const unsigned long long x = __shfl_sync(0xffffffffu, it, (k0 + a) & 31);
                if (live && k0 + a < count && key_of(x) < vocab) v[a].load(d_out + (uint64_t)(uint32_t)x * stride + col);
                if constexpr (ADD) {  // the row a run of equal tokens ends in, which no other warp writes: asked for along with the sums' rows
                    const uint32_t next = __shfl_sync(0xffffffffu, key_of(it), (k0 + a + 1) & 31);
                    if (live && k0 + a < count && key_of(x) < vocab && next != key_of(x)) old[a].load_coherent(d_table + (uint64_t)key_of(x) * hidden + col);
                }
            }
#pragma unroll
            for (int a = 0; a < AHEAD; a++) {
                const uint32_t k = k0 + a;
                const uint32_t key = __shfl_sync(0xffffffffu, key_of(it), k & 31), next = __shfl_sync(0xffffffffu, key_of(it), (k + 1) & 31);
                if (k >= count || key >= vocab) continue;
                if (live) {
#pragma unroll
                    for (int j = 0; j < N; j++) sum[j] += to_f32<T>(v[a].e[j]);
                }
                const bool ends = k + 1 < count ? next != key : !(c0 + count < n && next == key);
                if (!ends && k + 1 < count) continue;
                const bool left = begin == 0 && from_left;
                if (live) {
                    if (ends && !left) {
                        write_row<G, N>(d_table + (uint64_t)key * hidden + col, old[ADD ? a : 0], sum, scale, ADD);
                    } else {
                        float* c = carry + ((uint64_t)chunk * 2 + (left ? 0 : 1)) * hidden + col;
#pragma unroll
                        for (int j = 0; j < N; j++) c[j] = sum[j];
                    }
                }
#pragma unroll
                for (int j = 0; j < N; j++) sum[j] = 0.f;
                begin = k + 1;
            }
        }
    }
}

// ---- gradient, third launch: the tokens that cross chunks. The block of the chunk a token begins in adds the token's carries:
// its 8 warps take contiguous parts of the chunks, and the parts are added in order.
template <typename G, int N>
__global__ void __launch_bounds__(256) k_embed_join(const unsigned long long* __restrict__ sorted, uint32_t n, uint32_t vocab,
                                                    uint32_t hidden, G* d_table, const float* __restrict__ carry, float scale,
                                                    int accumulate, uint32_t* touched) {
    __shared__ float part[8][32 * N];
    let_next();
    after_previous();
    if (touched && blockIdx.y == 0)  // for the next call
        for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < ((uint64_t)vocab + 31) / 32; i += (uint64_t)gridDim.x * 256) touched[i] = 0;
    const uint32_t chunk = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const uint64_t c0 = (uint64_t)chunk * CHUNK, c1 = c0 + CHUNK;
    if (c1 >= n) return;  // nothing leaves the last chunk
    const uint32_t key = key_of(sorted[c1 - 1]), beyond = key_of(sorted[c1]), head = key_of(sorted[c0]), front = c0 > 0 ? key_of(sorted[c0 - 1]) : vocab;
    if (key >= vocab || beyond != key) return;
    if (head == key && front == key) return;  // began further left
    // the last chunk that begins with the token, 32 places asked at a time: it lies in [last, end)
    uint32_t last = chunk + 1, end = (uint32_t)(((uint64_t)n + CHUNK - 1) / CHUNK);
    while (end - last > 1) {
        const uint32_t step = (end - last + 31) / 32;
        const uint64_t probe = last + (uint64_t)(lane + 1) * step;
        const bool same = probe < end && key_of(sorted[probe * CHUNK]) == key;
        last += __popc(__ballot_sync(0xffffffffu, same)) * step;
        end = min(end, last + step);
    }
    const uint32_t parts = last - chunk;  // carries [0] of chunks chunk + 1 .. last
    const uint32_t col = blockIdx.y * 32 * N + lane * N;
    const uint32_t each = (parts + 7) / 8, p0 = min(parts, warp * each), p1 = min(parts, p0 + each);
    float sum[N];
#pragma unroll
    for (int j = 0; j < N; j++) sum[j] = 0.f;
    if (col < hidden) {
        if (warp == 0) {
#pragma unroll
            for (int j = 0; j < N; j++) sum[j] = carry[((uint64_t)chunk * 2 + 1) * hidden + col + j];
        }
#pragma unroll 4
        for (uint32_t p = p0; p < p1; p++) {
            const float* c = carry + (uint64_t)(chunk + 1 + p) * 2 * hidden + col;
#pragma unroll
            for (int j = 0; j < N; j++) sum[j] += c[j];
        }
    }
#pragma unroll
    for (int j = 0; j < N; j++) part[warp][lane * N + j] = sum[j];
    __syncthreads();
    if (warp || col >= hidden) return;
    for (int w = 1; w < 8; w++) {
#pragma unroll
        for (int j = 0; j < N; j++) sum[j] += part[w][lane * N + j];
    }
    write_row<G, N>(d_table + (uint64_t)key * hidden + col, sum, scale, accumulate != 0);
}

// Zeros over the rows without a token of one of `blocks` stretches of the table, by the block of that number. Up to FILL_ROWS rows at a
// time: the block marks the ones with a token in shared memory, then walks the stretch in aligned pieces of 32 bytes, whatever rows
// they lie in; a piece that a row with a token, or the stretch's end, cuts goes by elements.
constexpr uint32_t FILL_ROWS = 8192;
template <typename G>
__device__ void fill_without(const int64_t* __restrict__ ids, uint32_t n, uint32_t vocab, unsigned char* table, uint32_t row_bytes, uint32_t block, uint32_t blocks) {
    __shared__ uint32_t marks[FILL_ROWS / 32];
    const uint64_t per = ((uint64_t)vocab + blocks - 1) / blocks, r0 = min(block * per, (uint64_t)vocab), r1 = min(r0 + per, (uint64_t)vocab);
    const uint32_t at_once = min(FILL_ROWS, (1u << 31) / row_bytes);  // offsets within a stretch fit 32 bits
    const uint32_t zero[8] = {};
    for (uint64_t a = r0; a < r1; a += at_once) {
        const uint64_t b = min(a + at_once, r1);
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < FILL_ROWS / 32; i += blockDim.x) marks[i] = 0;
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < n; j += blockDim.x) {
            const int64_t id = ids[j];
            if (id >= (int64_t)a && id < (int64_t)b) atomicOr(&marks[(uint32_t)(id - a) >> 5], 1u << ((uint32_t)(id - a) & 31));
        }
        __syncthreads();
        auto marked = [&](uint32_t row) { return marks[row >> 5] >> (row & 31) & 1; };
        unsigned char* from = table + a * row_bytes;
        const uint32_t bytes = (uint32_t)(b - a) * row_bytes, skew = (uint32_t)(reinterpret_cast<uintptr_t>(from) & 31);
        const uint32_t pieces = (uint32_t)(((uint64_t)skew + bytes + 31) / 32);
        for (uint32_t p = threadIdx.x; p < pieces; p += blockDim.x) {
            const int64_t at = (int64_t)p * 32 - skew;  // of the piece, from the stretch's beginning
            const uint32_t begin = at < 0 ? 0 : (uint32_t)at, stop = (uint32_t)min(at + 32, (int64_t)bytes);
            uint32_t row = begin / row_bytes, row_end = (row + 1) * row_bytes;
            bool some = false, all = stop - begin == 32;  // rows without a token lie in the piece; nothing else does
            for (uint32_t r = row, end = row_end;; r++, end += row_bytes) {
                if (marked(r)) all = false;
                else some = true;
                if (end >= stop) break;
            }
            if (all) {
                store32(from + begin, zero);
            } else if (some) {
                for (uint32_t k = begin; k < stop; k += sizeof(G)) {
                    if (k == row_end) {
                        row++;
                        row_end += row_bytes;
                    }
                    if (!marked(row)) *reinterpret_cast<G*>(from + k) = from_f32<G>(0.f);
                }
            }
        }
    }
}

// ---- gradient of up to DIRECT tokens in one launch. A block has one token and up to 8 x 32 N columns (`across` blocks a token): it
// leaves where an equal id stands before the token; else it lists the equal ones behind, in order, and sums their rows, `splits` groups
// of warps a contiguous part of the list each, joined in order. The blocks behind write zeros to the rows without a token, where the
// table is overwritten: 590 x 128 bf16 of 4131 rows 4.6 us, 6.0 with a fill of the whole table in front; 786 x 837 f16 of 113836 rows 42 and
// 43.5.
template <typename T, typename G, int N>
__global__ void __launch_bounds__(256) k_embed_direct(const int64_t* __restrict__ ids, uint32_t n, uint32_t vocab, const T* __restrict__ d_out,
                                                      uint64_t stride, uint32_t hidden, G* d_table, float scale, int accumulate, uint32_t wide,
                                                      uint32_t across) {
    __shared__ uint16_t list[DIRECT];
    __shared__ uint32_t counts[8];
    __shared__ float share[256 * N];
    if (blockIdx.x >= n * across) {
        fill_without<G>(ids, n, vocab, reinterpret_cast<unsigned char*>(d_table), hidden * (uint32_t)sizeof(G), blockIdx.x - n * across, gridDim.x - n * across);
        return;
    }
    const uint32_t i = blockIdx.x / across, warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int64_t id = ids[i];
    if ((uint64_t)id >= vocab) return;
    bool before = false;
    for (uint32_t j = threadIdx.x; j < i; j += 256) before |= ids[j] == id;
    if (__syncthreads_or(before)) return;
    // the equal ones from i on: each warp a run of 32 x turns tokens
    const uint32_t turns = (n - i + 255) / 256, begin = i + warp * turns * 32;
    uint32_t count = 0;
    for (uint32_t t = 0; t < turns; t++) {
        const uint32_t j = begin + t * 32 + lane;
        count += __popc(__ballot_sync(0xffffffffu, j < n && ids[j] == id));
    }
    if (lane == 0) counts[warp] = count;
    __syncthreads();
    uint32_t at = 0, total = 0;
    for (uint32_t w = 0; w < 8; w++) {
        at += w < warp ? counts[w] : 0;
        total += counts[w];
    }
    for (uint32_t t = 0; t < turns; t++) {
        const uint32_t j = begin + t * 32 + lane;
        const bool yes = j < n && ids[j] == id;
        const uint32_t bits = __ballot_sync(0xffffffffu, yes);
        if (yes) list[at + __popc(bits & ((1u << lane) - 1))] = (uint16_t)j;
        at += __popc(bits);
    }
    __syncthreads();
    // `wide` warps along a row, 8 / wide along the list
    const uint32_t splits = 8 / wide, part = warp / wide, col = ((blockIdx.x - i * across) * wide + warp % wide) * 32 * N + lane * N;
    const bool live = part < splits && col < hidden;
    float sum[N];
#pragma unroll
    for (int j = 0; j < N; j++) sum[j] = 0.f;
    if (live) {
        const uint32_t each = (total + splits - 1) / splits, k0 = min(total, part * each), k1 = min(total, k0 + each);
        constexpr int AHEAD = 8;
        for (uint32_t k = k0; k < k1; k += AHEAD) {
            Vec<T, N> v[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; a++)
                if (k + a < k1) v[a].load(d_out + (uint64_t)list[k + a] * stride + col);
#pragma unroll
            for (int a = 0; a < AHEAD; a++)
                if (k + a < k1) {
#pragma unroll
                    for (int j = 0; j < N; j++) sum[j] += to_f32<T>(v[a].e[j]);
                }
        }
    }
    if (splits > 1) {
#pragma unroll
        for (int j = 0; j < N; j++) share[threadIdx.x * N + j] = sum[j];
        __syncthreads();
        if (part) return;
        for (uint32_t p = 1; p < splits; p++)
#pragma unroll
            for (int j = 0; j < N; j++) sum[j] += share[(p * wide * 32 + threadIdx.x) * N + j];
    }
    if (live) write_row<G, N>(d_table + (uint64_t)id * hidden + col, sum, scale, accumulate != 0);
}

uint64_t mark_bytes(const oxz_embed_desc& d) { return (d.vocab + 31) / 32 * 4; }

// From the first launch of a call that marks rows to the last, which takes the marks away. A call that breaks off in between clears them
// itself: the next call relies on it, and so do graphs captured before. (A captured call runs nothing now and changes nothing.)
struct Marking {
    oxz_embed* e;
    cudaStream_t s;
    bool open = false;
    void close() {
        if (open) e->clean = true;
        open = false;
    }
    ~Marking() {
        if (!open) return;
        e->clean = cudaMemsetAsync(e->touched, 0, mark_bytes(e->d), s) == cudaSuccess;
        if (!e->clean) (void)cudaGetLastError();
    }
};

bool misaligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) % to) != 0; }

template <typename T, int N>
int32_t lookup(const oxz_embed_desc& d, const int64_t* ids, uint64_t n, const void* table, void* out, uint64_t stride, cudaStream_t s) {
    const uint32_t pieces = (uint32_t)((d.hidden + 128 * N - 1) / (128 * N));
    const uint64_t blocks = std::min<uint64_t>((n * pieces + 7) / 8, 1u << 30);
    OXZ_CUDA(launch_after(false, k_embed_lookup<T, N>, (unsigned)blocks, 256, 0, s, ids, n, static_cast<const T*>(table), static_cast<T*>(out), stride,
                          (uint32_t)d.hidden, d.vocab, (float)d.scale, pieces));
    return OXZ_OK;
}

template <typename T, typename G, int N>
int32_t sums(oxz_embed* e, uint32_t n, const int64_t* ids, const unsigned long long* sorted, const void* d_out, uint64_t stride, void* d_table,
             int32_t accumulate, cudaStream_t s) {
    const oxz_embed_desc& d = e->d;
    const uint32_t slices = (uint32_t)((d.hidden + 32 * N - 1) / (32 * N)), vocab = (uint32_t)d.vocab, hidden = (uint32_t)d.hidden;
    if (n <= DIRECT) {
        const uint32_t wide = std::min<uint32_t>(8, slices), across = (slices + wide - 1) / wide;
        const uint64_t bytes = d.vocab * d.hidden * sizeof(G);
        const unsigned fillers = accumulate ? 0 : (unsigned)std::min<uint64_t>(e->sms * 8, (bytes + (16 << 10) - 1) / (16 << 10));
        OXZ_CUDA(launch_after(false, k_embed_direct<T, G, N>, n * across + fillers, 256, 0, s, ids, n, vocab, static_cast<const T*>(d_out), stride, hidden,
                              static_cast<G*>(d_table), (float)d.scale, accumulate, wide, across));
        return OXZ_OK;
    }
    const uint32_t chunks = (n + CHUNK - 1) / CHUNK;
    const unsigned blocks = (unsigned)std::min<uint64_t>(((uint64_t)chunks * slices + 7) / 8, 1u << 30);
    uint32_t* touched = accumulate ? nullptr : e->touched;
    const unsigned fillers = accumulate ? 0 : (unsigned)std::min<uint64_t>(e->sms * 8, (d.vocab + 7) / 8);
    OXZ_CUDA(launch_after(true, accumulate ? k_embed_sums<T, G, N, true> : k_embed_sums<T, G, N, false>, blocks + fillers, 256, 0, s, sorted, n, vocab,
                          static_cast<const T*>(d_out), stride, hidden, static_cast<G*>(d_table), e->carry, (float)d.scale, slices, blocks, touched));
    OXZ_CUDA(launch_after(true, k_embed_join<G, N>, dim3(chunks - 1, slices), 256, 0, s, sorted, n, vocab, hidden, static_cast<G*>(d_table), e->carry,
                          (float)d.scale, accumulate, touched));
    return OXZ_OK;
}

}  // namespace
}  // namespace oxz

using namespace oxz;

extern "C" {

int32_t oxz_embed_create(const oxz_embed_desc* desc, oxz_embed** out) {
    return guarded("oxz_embed_create", [&]() -> int32_t {
        if (!desc || !out) return fail(OXZ_ERR_INVALID, "oxz_embed_create: null argument");
        *out = nullptr;
        const oxz_embed_desc& d = *desc;
        if (d.max_tokens == 0 || d.max_tokens > 0x7fffffffull)
            return fail(OXZ_ERR_INVALID, "oxz_embed_create: max_tokens %llu is outside 1..2^31-1", (unsigned long long)d.max_tokens);
        if (d.vocab == 0 || d.vocab > 0x7fffffffull)
            return fail(OXZ_ERR_INVALID, "oxz_embed_create: vocab %llu is outside 1..2^31-1", (unsigned long long)d.vocab);
        if (d.hidden == 0 || d.hidden > (1u << 20))
            return fail(OXZ_ERR_INVALID, "oxz_embed_create: hidden %llu is outside 1..2^20", (unsigned long long)d.hidden);
        if (!std::isfinite((float)d.scale)) return fail(OXZ_ERR_INVALID, "oxz_embed_create: scale %g is not a finite f32", d.scale);
        if (d.dtype != OXZ_F32 && d.dtype != OXZ_BF16 && d.dtype != OXZ_F16)
            return fail(OXZ_ERR_INVALID, "oxz_embed_create: dtype %d is none of f32, bf16, f16", d.dtype);
        if (d.grad_dtype != d.dtype && d.grad_dtype != OXZ_F32)
            return fail(OXZ_ERR_INVALID, "oxz_embed_create: grad_dtype %d is neither the dtype (%d) nor f32", d.grad_dtype, d.dtype);
        if (d.device < 0) return fail(OXZ_ERR_INVALID, "oxz_embed_create: device %d", d.device);
        oxz_embed* e = new oxz_embed();
        e->d = d;
        *out = e;
        return OXZ_OK;
    });
}

int32_t oxz_embed_alloc(oxz_embed* e, uint64_t* workspace_bytes) {
    return guarded("oxz_embed_alloc", [&]() -> int32_t {
        if (!e) return fail(OXZ_ERR_INVALID, "oxz_embed_alloc: null handle");
        if (!e->allocated) {
            DeviceGuard dev;
            OXZ_TRY(dev.enter(e->d.device));
            const uint64_t chunks = (e->d.max_tokens + CHUNK - 1) / CHUNK;
            const uint64_t items = e->d.max_tokens * 8, carry = chunks * 2 * e->d.hidden * 4;
            // what a failed attempt left behind is kept and used by the next one
            for (int i = 0; i < 2; i++)
                if (!e->sorted[i]) OXZ_CUDA(cudaMalloc((void**)&e->sorted[i], items));
            if (!e->carry) OXZ_CUDA(cudaMalloc((void**)&e->carry, carry));
            if (!e->touched) OXZ_CUDA(cudaMalloc((void**)&e->touched, mark_bytes(e->d)));
            OXZ_CUDA(cudaMemset(e->touched, 0, mark_bytes(e->d)));
            OXZ_CUDA(cudaDeviceSynchronize());
            e->clean = true;
            OXZ_CUDA(cudaDeviceGetAttribute(&e->sms, cudaDevAttrMultiProcessorCount, e->d.device));
            OXZ_TRY(e->order.create());
            OXZ_CUDA(cudaFuncSetAttribute(k_embed_sort, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SortShared)));
            e->bytes = 2 * items + carry + mark_bytes(e->d);
            e->allocated = true;
        }
        if (workspace_bytes) *workspace_bytes = e->bytes;
        return OXZ_OK;
    });
}

int32_t oxz_embed_destroy(oxz_embed* e) {
    return guarded("oxz_embed_destroy", [&]() -> int32_t {
        if (!e) return OXZ_OK;
        DeviceGuard dev;
        if (e->sorted[0] || e->carry) dev.enter(e->d.device);
        e->order.destroy();
        for (int i = 0; i < 2; i++)
            if (e->sorted[i]) cudaFree(e->sorted[i]);
        if (e->carry) cudaFree(e->carry);
        if (e->touched) cudaFree(e->touched);
        delete e;
        return OXZ_OK;
    });
}

int32_t oxz_embed_lookup_async(const oxz_embed* e, const int64_t* ids, uint64_t n, const void* table, void* out, uint64_t out_stride,
                               void* stream) {
    return guarded("oxz_embed_lookup_async", [&]() -> int32_t {
        if (!e) return fail(OXZ_ERR_INVALID, "oxz_embed_lookup_async: null handle");
        if (n == 0) return OXZ_OK;
        if (!ids || !table || !out) return fail(OXZ_ERR_INVALID, "oxz_embed_lookup_async: null argument");
        const oxz_embed_desc& d = e->d;
        if (n > d.max_tokens)
            return fail(OXZ_ERR_INVALID, "oxz_embed_lookup_async: %llu tokens, the handle was made for %llu", (unsigned long long)n, (unsigned long long)d.max_tokens);
        if (out_stride == 0) out_stride = d.hidden;
        if (out_stride < d.hidden || out_stride > (1ull << 31))
            return fail(OXZ_ERR_INVALID, "oxz_embed_lookup_async: out_stride %llu with rows of %llu", (unsigned long long)out_stride, (unsigned long long)d.hidden);
        const size_t es = dtype_size(d.dtype);
        if (misaligned(ids, 8) || misaligned(table, es) || misaligned(out, es))
            return fail(OXZ_ERR_INVALID, "oxz_embed_lookup_async: a pointer is not aligned to its element");
        DeviceGuard dev;
        OXZ_TRY(dev.enter(d.device));
        cudaStream_t s = (cudaStream_t)stream;
        const bool wide = !misaligned(table, 16) && !misaligned(out, 16) && d.hidden * es % 16 == 0 && out_stride * es % 16 == 0;
        if (d.dtype == OXZ_F32) return wide ? lookup<float, 4>(d, ids, n, table, out, out_stride, s) : lookup<float, 1>(d, ids, n, table, out, out_stride, s);
        if (d.dtype == OXZ_BF16) return wide ? lookup<__nv_bfloat16, 8>(d, ids, n, table, out, out_stride, s) : lookup<__nv_bfloat16, 1>(d, ids, n, table, out, out_stride, s);
        return wide ? lookup<__half, 8>(d, ids, n, table, out, out_stride, s) : lookup<__half, 1>(d, ids, n, table, out, out_stride, s);
    });
}

int32_t oxz_embed_grads_async(oxz_embed* e, const int64_t* ids, uint64_t n, const void* d_out, uint64_t d_out_stride, void* d_table,
                              int32_t accumulate, void* stream) {
    return guarded("oxz_embed_grads_async", [&]() -> int32_t {
        if (!e) return fail(OXZ_ERR_INVALID, "oxz_embed_grads_async: null handle");
        const oxz_embed_desc& d = e->d;
        if (!d_table || (n && (!ids || !d_out))) return fail(OXZ_ERR_INVALID, "oxz_embed_grads_async: null argument");
        if (n > d.max_tokens)
            return fail(OXZ_ERR_INVALID, "oxz_embed_grads_async: %llu tokens, the handle was made for %llu", (unsigned long long)n, (unsigned long long)d.max_tokens);
        if (d_out_stride == 0) d_out_stride = d.hidden;
        if (d_out_stride < d.hidden || d_out_stride > (1ull << 31))
            return fail(OXZ_ERR_INVALID, "oxz_embed_grads_async: d_out_stride %llu with rows of %llu", (unsigned long long)d_out_stride, (unsigned long long)d.hidden);
        const size_t es = dtype_size(d.dtype), gs = dtype_size(d.grad_dtype);
        if (misaligned(ids, 8) || misaligned(d_out, es) || misaligned(d_table, gs))
            return fail(OXZ_ERR_INVALID, "oxz_embed_grads_async: a pointer is not aligned to its element");
        if (!e->allocated) return fail(OXZ_ERR_STATE, "oxz_embed_grads_async: no workspace: call oxz_embed_alloc first");
        if (n == 0 && accumulate) return OXZ_OK;
        DeviceGuard dev;
        OXZ_TRY(dev.enter(d.device));
        cudaStream_t s = (cudaStream_t)stream;
        Turn turn(e->order);
        OXZ_TRY(turn.begin(s));
        const unsigned long long* sorted = e->sorted[0];
        uint32_t* touched = accumulate ? nullptr : e->touched;
        Marking marking{e, s};
        if (n > DIRECT) {
            if (touched && !e->clean) OXZ_CUDA(cudaMemsetAsync(touched, 0, mark_bytes(d), s));
            marking.open = touched && !turn.captured();
            if (n <= RANKED) {
                const uint32_t tokens = std::min<uint32_t>(64, ((uint32_t)n + e->sms - 1) / e->sms), parts = tokens <= 32 ? 32 : 16;
                OXZ_CUDA(launch_after(false, parts == 32 ? k_embed_rank<32> : k_embed_rank<16>, ((unsigned)n + tokens - 1) / tokens, (tokens * parts + 31) / 32 * 32, 0,
                                      s, ids, (uint32_t)n, (uint32_t)d.vocab, tokens, e->sorted[0], touched));
            } else {
                // keys run to vocab itself (ids outside the table): as few passes of at most DIGIT_BITS bits as hold them, of equal width
                int key_bits = 1;
                while ((d.vocab >> key_bits) != 0) key_bits++;
                const int passes = (key_bits + DIGIT_BITS - 1) / DIGIT_BITS, bits = (key_bits + passes - 1) / passes;
                sorted = e->sorted[passes & 1];
                cudaLaunchConfig_t cfg{};
                cfg.gridDim = dim3(SORT_CLUSTER);
                cfg.blockDim = dim3(SORT_THREADS);
                cfg.dynamicSmemBytes = sizeof(SortShared);
                cfg.stream = s;
                cudaLaunchAttribute attr{};
                attr.id = cudaLaunchAttributeClusterDimension;
                attr.val.clusterDim = {SORT_CLUSTER, 1, 1};
                cfg.attrs = &attr;
                cfg.numAttrs = 1;
                OXZ_CUDA(cudaLaunchKernelEx(&cfg, k_embed_sort, ids, (uint32_t)n, (uint32_t)d.vocab, passes, bits, e->sorted[0], e->sorted[1], touched));
            }
        }
        {
            const bool wide = !misaligned(d_out, 16) && !misaligned(d_table, 16) && d.hidden * es % 16 == 0 && d_out_stride * es % 16 == 0;
            const uint32_t m = (uint32_t)n;
            const uint64_t st = d_out_stride;
            const bool f32g = d.grad_dtype == OXZ_F32;
            if (d.dtype == OXZ_F32) OXZ_TRY((wide ? sums<float, float, 4>(e, m, ids, sorted, d_out, st, d_table, accumulate, s) : sums<float, float, 1>(e, m, ids, sorted, d_out, st, d_table, accumulate, s)));
            else if (d.dtype == OXZ_BF16 && !f32g) OXZ_TRY((wide ? sums<__nv_bfloat16, __nv_bfloat16, 8>(e, m, ids, sorted, d_out, st, d_table, accumulate, s) : sums<__nv_bfloat16, __nv_bfloat16, 1>(e, m, ids, sorted, d_out, st, d_table, accumulate, s)));
            else if (d.dtype == OXZ_BF16) OXZ_TRY((wide ? sums<__nv_bfloat16, float, 8>(e, m, ids, sorted, d_out, st, d_table, accumulate, s) : sums<__nv_bfloat16, float, 1>(e, m, ids, sorted, d_out, st, d_table, accumulate, s)));
            else if (!f32g) OXZ_TRY((wide ? sums<__half, __half, 8>(e, m, ids, sorted, d_out, st, d_table, accumulate, s) : sums<__half, __half, 1>(e, m, ids, sorted, d_out, st, d_table, accumulate, s)));
            else OXZ_TRY((wide ? sums<__half, float, 8>(e, m, ids, sorted, d_out, st, d_table, accumulate, s) : sums<__half, float, 1>(e, m, ids, sorted, d_out, st, d_table, accumulate, s)));
        }
        marking.close();
        return turn.end();
    });
}

}  // extern "C"
