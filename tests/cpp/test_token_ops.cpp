// The C++ mirror's token operators: refusals without a GPU, and one small call of each with --gpu.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include <cuda_runtime.h>

#include "../../oxidizr_b200/cpp/oxz.hpp"

using namespace oxidizr;

static int failures = 0;
#define EXPECT(c)                                                  \
    do {                                                           \
        if (!(c)) {                                                \
            std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #c); \
            failures++;                                            \
        }                                                          \
    } while (0)

template <typename F>
static bool refused(F&& f, int32_t status, const char* text) {
    try {
        f();
    } catch (const Error& e) {
        return e.status == status && std::strstr(e.what(), text) != nullptr;
    }
    return false;
}

static void host_only() {
    EXPECT(refused([] { TokenEmbedding(0, 8, 4, OXZ_BF16, OXZ_BF16); }, OXZ_ERR_INVALID, "vocab 0"));
    EXPECT(refused([] { LossHead(10, 8, 0, OXZ_BF16, OXZ_BF16); }, OXZ_ERR_INVALID, "max_rows 0"));
    EXPECT(refused([] { LossHead(10, 8, 4, OXZ_F32, OXZ_BF16); }, OXZ_ERR_INVALID, "grad_dtype"));
    LossHead head(10, 8, 4, OXZ_F32, OXZ_F32);
    alignas(16) float some[16];
    alignas(8) int64_t targets[2];
    const oxz_head_batch b{2, some, 0, some, targets, nullptr};
    EXPECT(refused([&] { head.loss(b, nullptr, nullptr, nullptr); }, OXZ_ERR_STATE, "oxz_head_alloc"));
    TokenEmbedding emb(10, 8, 4, OXZ_F32, OXZ_F32);
    EXPECT(refused([&] { emb.grads(targets, 2, some, some, false); }, OXZ_ERR_STATE, "oxz_embed_alloc"));
    EXPECT(refused([&] { emb.lookup(targets, 5, some, some); }, OXZ_ERR_INVALID, "5 tokens"));
}

template <typename T>
static T* device(const std::vector<T>& v) {
    T* p = nullptr;
    EXPECT(cudaMalloc(&p, v.size() * sizeof(T)) == cudaSuccess);
    EXPECT(cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice) == cudaSuccess);
    return p;
}
template <typename T>
static std::vector<T> host(const T* p, size_t n) {
    std::vector<T> v(n);
    EXPECT(cudaMemcpy(v.data(), p, n * sizeof(T), cudaMemcpyDeviceToHost) == cudaSuccess);
    return v;
}

static void on_gpu() {
    // two words, one hidden element: logits x w_v, the loss log(1 + exp(x (w_other - w_target)))
    const uint64_t V = 2, H = 4, N = 3;
    const std::vector<float> table{1, 0, 0, 0, 0, 2, 0, 0};
    const std::vector<int64_t> ids{0, 1, 0}, targets{0, 0, 1};
    float* w = device(table);
    int64_t *d_ids = device(ids), *d_t = device(targets);
    float *x = device(std::vector<float>(N * H)), *dx = device(std::vector<float>(N * H)), *dw = device(std::vector<float>(V * H));
    float *loss = device(std::vector<float>(N)), *totals = device(std::vector<float>(2));
    TokenEmbedding emb(V, H, N, OXZ_F32, OXZ_F32, 3.0);
    EXPECT(emb.alloc() > 0);
    emb.lookup(d_ids, N, w, x);
    EXPECT(cudaDeviceSynchronize() == cudaSuccess);
    EXPECT((host(x, N * H) == std::vector<float>{3, 0, 0, 0, 0, 6, 0, 0, 3, 0, 0, 0}));
    LossHead head(V, H, N, OXZ_F32, OXZ_F32);
    EXPECT(head.alloc() > 0);
    const oxz_head_batch b{N, x, 0, w, d_t, nullptr};
    const oxz_head_grads g{dx, 0, dw, 1.0, 0, 0};
    head.loss_and_grads(b, loss, nullptr, totals, g);
    emb.grads(d_ids, N, dx, dw, true);
    EXPECT(cudaDeviceSynchronize() == cudaSuccess);
    // logits of the rows: (3, 0), (0, 12), (3, 0)
    const double want[3] = {std::log1p(std::exp(-3.0)), 12.0 + std::log1p(std::exp(-12.0)), 3.0 + std::log1p(std::exp(-3.0))};
    const auto got = host(loss, N);
    double sum = 0;
    for (int i = 0; i < 3; i++) {
        sum += want[i];
        EXPECT(std::fabs(got[i] - want[i]) <= 1e-5);
    }
    const auto t = host(totals, 2);
    EXPECT(std::fabs(t[0] - sum) <= 1e-5 * sum && t[1] == 3.0f);
    // G = p - y; the tied gradient G^T x + 3 * (G w scattered to the ids)
    const double p3 = 1 / (1 + std::exp(-3.0)), p12 = 1 / (1 + std::exp(-12.0));
    const double G[3][2] = {{p3 - 1, 1 - p3}, {(1 - p12) - 1, p12}, {p3, (1 - p3) - 1}};
    const double X[3][4] = {{3, 0, 0, 0}, {0, 6, 0, 0}, {3, 0, 0, 0}};
    double D[2][4] = {};
    for (int i = 0; i < 3; i++)
        for (int v = 0; v < 2; v++)
            for (int k = 0; k < 4; k++) {
                D[v][k] += G[i][v] * X[i][k];
                D[ids[i]][k] += 3.0 * G[i][v] * table[v * 4 + k];
            }
    const auto d = host(dw, V * H);
    for (int e = 0; e < 8; e++) EXPECT(std::fabs(d[e] - D[e / 4][e % 4]) <= 1e-5 * 20);
    for (void* q : {(void*)w, (void*)d_ids, (void*)d_t, (void*)x, (void*)dx, (void*)dw, (void*)loss, (void*)totals}) cudaFree(q);
}

int main(int argc, char** argv) {
    host_only();
    if (argc > 1 && std::strcmp(argv[1], "--gpu") == 0) on_gpu();
    std::printf(failures ? "%d failed\n" : "all passed\n", failures);
    return failures != 0;
}
