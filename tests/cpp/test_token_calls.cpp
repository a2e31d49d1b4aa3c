// The token operators' calls on the host, over a runtime of notes (fake_cuda.hpp): what they enqueue, in what order, and what is left
// when one of the runtime's calls fails in the middle.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <functional>
#include <thread>

#include "../../include/oxz_dpstep.h"
#include "fake_cuda.hpp"

static std::atomic<int> failures{0};
#define EXPECT(c, ...)                                                          \
    do {                                                                        \
        if (!(c)) {                                                             \
            std::printf("FAILED %s:%d: %s ", __FILE__, __LINE__, #c);           \
            std::printf(" " __VA_ARGS__);                                       \
            std::printf("\n");                                                  \
            failures++;                                                         \
        }                                                                       \
    } while (0)

static const cudaStream_t A = (cudaStream_t)0x1000, B = (cudaStream_t)0x2000, C = (cudaStream_t)0x3000;
static void* const p = (void*)(1 << 20);  // an address that no kernel reads here

// A handle and the call it is tested with
struct Operator {
    const char* name;
    std::function<void*()> make;
    std::function<int32_t(void*, cudaStream_t)> call;
    std::function<void(void*)> destroy;
};

static void* embed(uint64_t tokens) {
    const oxz_embed_desc d{tokens, 64, 1000, 1.0, OXZ_BF16, OXZ_BF16, 0, 0};
    oxz_embed* e = nullptr;
    EXPECT(oxz_embed_create(&d, &e) == OXZ_OK);
    EXPECT(oxz_embed_alloc(e, nullptr) == OXZ_OK);
    return e;
}
static void* head(uint64_t rows, uint64_t vocab, uint64_t piece_bytes) {
    const oxz_head_desc d{rows, 64, vocab, piece_bytes, OXZ_BF16, OXZ_BF16, 0, 0};
    oxz_head* h = nullptr;
    EXPECT(oxz_head_create(&d, &h) == OXZ_OK);
    EXPECT(oxz_head_alloc(h, nullptr) == OXZ_OK);
    return h;
}
static Operator embed_grads(const char* name, uint64_t n, int accumulate) {
    return {name, [=] { return embed(n); },
            [=](void* h, cudaStream_t s) { return oxz_embed_grads_async((oxz_embed*)h, (const int64_t*)p, n, p, 0, p, accumulate, s); },
            [](void* h) { oxz_embed_destroy((oxz_embed*)h); }};
}
static Operator head_train(const char* name, uint64_t rows, uint64_t vocab, uint64_t piece_bytes) {
    return {name, [=] { return head(rows, vocab, piece_bytes); },
            [=](void* h, cudaStream_t s) {
                const oxz_head_batch b{rows, p, 0, p, (const int64_t*)p, nullptr};
                const oxz_head_grads g{p, 0, p, 1.0, 0, 0};
                return oxz_head_loss_grads_async((oxz_head*)h, &b, (float*)p, (float*)p, (float*)p, &g, s);
            },
            [](void* h) { oxz_head_destroy((oxz_head*)h); }};
}
static std::vector<Operator> operators() {
    return {embed_grads("embed 100", 100, 0), embed_grads("embed 2000", 2000, 0), embed_grads("embed 9000", 9000, 0), embed_grads("embed 9000 added", 9000, 1),
            head_train("head 5", 5, 500, 0), head_train("head 40", 40, 500, 0), head_train("head 2000 in pieces", 2000, 3000, 1)};
}
// An error is the failing call's: what runs after it is not refused for it, on the same handle or another.
static void an_error_is_reported_once() {
    for (const Operator& op : operators()) {
        void* h = op.make();
        fake::memory = 1 << 10;
        const oxz_head_desc d{40, 64, 500, 0, OXZ_F32, OXZ_F32, 0, 0};
        oxz_head* large = nullptr;
        EXPECT(oxz_head_create(&d, &large) == OXZ_OK);
        EXPECT(oxz_head_alloc(large, nullptr) == OXZ_ERR_CUDA);
        oxz_head_destroy(large);
        fake::memory = ~size_t(0);
        EXPECT(op.call(h, A) == OXZ_OK, "%s: %s", op.name, fake::message.c_str());
        fake::last = cudaErrorInvalidValue;  // what some other part of the program left
        EXPECT(op.call(h, A) == OXZ_OK, "%s: %s", op.name, fake::message.c_str());
        fake::last = cudaSuccess;
        fake::fail_at = 1;  // the first launch
        EXPECT(op.call(h, A) == OXZ_ERR_CUDA, "%s", op.name);
        EXPECT(op.call(h, A) == OXZ_OK, "%s: %s", op.name, fake::message.c_str());
        op.destroy(h);
    }
    const oxz_embed_desc d{8, 64, 1000, 1.0, OXZ_BF16, OXZ_BF16, 0, 0};
    oxz_embed* e = nullptr;
    EXPECT(oxz_embed_create(&d, &e) == OXZ_OK);
    fake::last = cudaErrorInvalidValue;
    EXPECT(oxz_embed_lookup_async(e, (const int64_t*)p, 8, p, p, 0, A) == OXZ_OK, "%s", fake::message.c_str());
    fake::fail_at = 0;
    EXPECT(oxz_embed_lookup_async(e, (const int64_t*)p, 8, p, p, 0, A) == OXZ_ERR_CUDA);
    EXPECT(oxz_embed_lookup_async(e, (const int64_t*)p, 8, p, p, 0, A) == OXZ_OK, "%s", fake::message.c_str());
    fake::last = cudaSuccess;
    oxz_embed_destroy(e);
}

static bool works(const fake::Op& o) { return o.kind == fake::LAUNCH || o.kind == fake::CLEAR; }

// A call that breaks off has launched kernels that use the handle's workspace: the next call, on another stream, waits for them.
static void the_next_call_waits_for_one_that_broke_off() {
    for (const Operator& op : operators()) {
        for (int k = 0;; k++) {
            void* h = op.make();
            EXPECT(op.call(h, A) == OXZ_OK, "%s", op.name);
            fake::ops.clear();
            fake::fail_at = k;
            const int32_t rc = op.call(h, A);
            const bool reached = fake::fail_at < 0;
            fake::fail_at = -1;
            if (!reached) {
                EXPECT(rc == OXZ_OK && k > 2, "%s: %d calls", op.name, k);
                op.destroy(h);
                break;
            }
            EXPECT(rc == OXZ_ERR_CUDA, "%s: call %d failed", op.name, k);
            int work = -1, record = -1;
            for (int i = 0; i < (int)fake::ops.size(); i++) {
                if (works(fake::ops[i])) work = i;
                if (fake::ops[i].kind == fake::RECORD) record = i;
            }
            const size_t before = fake::ops.size();
            EXPECT(op.call(h, B) == OXZ_OK, "%s: after call %d failed: %s", op.name, k, fake::message.c_str());
            if (work >= 0 && rc != OXZ_OK) {
                EXPECT(record > work, "%s: call %d failed, nothing marks the end of what was launched", op.name, k);
                EXPECT(fake::ops[before].kind == fake::WAIT && fake::ops[before].stream == B && record >= 0 && fake::ops[before].what == fake::ops[record].what,
                       "%s: call %d failed, the next does not wait", op.name, k);
            }
            op.destroy(h);
        }
    }
}

// Where what is done about a failure fails as well, the first one is reported.
static void the_first_failure_is_the_one_reported() {
    for (const Operator& op : operators()) {
        void* h = op.make();
        EXPECT(op.call(h, A) == OXZ_OK);
        fake::fail_at = 1;  // the first launch, and all that follows
        fake::fail_for = 1000;
        EXPECT(op.call(h, A) == OXZ_ERR_CUDA);
        EXPECT(fake::message.find("launch_after") == 0 || fake::message.find("cudaLaunchKernelEx") == 0, "%s: %s", op.name, fake::message.c_str());
        fake::fail_at = -1;
        fake::fail_for = 1;
        EXPECT(op.call(h, A) == OXZ_OK, "%s: %s", op.name, fake::message.c_str());
        op.destroy(h);
    }
}

// The gradient that writes its table marks the rows that have a token, and its last kernel takes the marks away. A call that breaks off
// between the two leaves marks: rows that the next call, or the replay of an older graph, would take for written.
static void marks_are_taken_away_after_a_call_that_broke_off() {
    const Operator op = embed_grads("embed 2000", 2000, 0);
    for (int k : {2, 3}) {  // after the wait and the marks: the sums, or the kernel that takes the marks away
        void* h = op.make();
        EXPECT(op.call(h, A) == OXZ_OK);
        // at once, for graphs that were captured while there were none
        fake::ops.clear();
        fake::fail_at = k;
        EXPECT(op.call(h, A) == OXZ_ERR_CUDA);
        int launch = -1, clear = -1;
        for (int i = 0; i < (int)fake::ops.size(); i++) {
            if (fake::ops[i].kind == fake::LAUNCH) launch = i;
            if (fake::ops[i].kind == fake::CLEAR) clear = i;
        }
        EXPECT(launch >= 0 && clear > launch, "call %d failed, launches up to %d, marks cleared at %d", k, launch, clear);
        // where that fails too: before the next call that runs, however many were captured meanwhile, and within each of those
        fake::fail_at = k;
        fake::fail_for = 2;
        EXPECT(op.call(h, A) == OXZ_ERR_CUDA);
        fake::capturing.insert(C);
        for (int i = 0; i < 2; i++) {
            fake::ops.clear();
            EXPECT(op.call(h, C) == OXZ_OK);
            EXPECT(!fake::ops.empty() && fake::ops[0].kind == fake::CLEAR && fake::ops[0].captured, "captured call %d", i);
        }
        fake::capturing.clear();
        fake::ops.clear();
        EXPECT(op.call(h, B) == OXZ_OK);
        size_t first = 0;
        while (first < fake::ops.size() && !works(fake::ops[first])) first++;
        EXPECT(first < fake::ops.size() && fake::ops[first].kind == fake::CLEAR, "call %d failed, captures, then a call over old marks", k);
        // and not again
        fake::ops.clear();
        EXPECT(op.call(h, B) == OXZ_OK);
        for (const fake::Op& o : fake::ops) EXPECT(o.kind != fake::CLEAR);
        op.destroy(h);
    }
    // a capture that breaks off has run nothing
    void* h = op.make();
    fake::capturing.insert(C);
    fake::fail_at = 1;
    EXPECT(op.call(h, C) == OXZ_ERR_CUDA);
    fake::capturing.clear();
    fake::ops.clear();
    EXPECT(op.call(h, A) == OXZ_OK);
    for (const fake::Op& o : fake::ops) EXPECT(o.kind != fake::CLEAR);
    op.destroy(h);
}

// Threads with a handle each share nothing that one of them writes: the thread sanitizer watches.
static void threads_with_a_handle_each() {
    for (const Operator& op : operators()) {
        std::vector<std::thread> threads;
        std::atomic<int> ready{0};
        for (int k = 0; k < 4; k++)
            threads.emplace_back([&, k] {
                void* h = op.make();
                ready++;
                while (ready < 4) std::this_thread::yield();
                for (int i = 0; i < 3; i++) EXPECT(op.call(h, (cudaStream_t)(uintptr_t)(0x10000 + 16 * k)) == OXZ_OK, "%s", op.name);
                op.destroy(h);
            });
        for (std::thread& t : threads) t.join();
    }
}

// A head whose every batch streams the weight has no workspace for tiles; one that may meet another batch has both.
static void a_handful_of_rows_takes_no_workspace_for_tiles() {
    const struct { uint64_t rows, hidden, vocab; int32_t dtype, grad; bool streams; } cases[] = {
        {1, 512, 100315, OXZ_F32, OXZ_F32, true},    {16, 768, 39380, OXZ_F32, OXZ_F32, true},    {8, 1024, 32000, OXZ_BF16, OXZ_BF16, true},
        {4, 5760, 32000, OXZ_F16, OXZ_F32, true},    {8, 345, 20000, OXZ_F16, OXZ_F16, true},     {16, 345, 3000, OXZ_BF16, OXZ_BF16, true},
        {17, 512, 32000, OXZ_F32, OXZ_F32, false},   {16, 1024, 32000, OXZ_BF16, OXZ_BF16, false},  // a batch off 16 bytes would go by tiles
        {8, 5768, 32000, OXZ_BF16, OXZ_BF16, false}, {16, 2436, 32000, OXZ_F32, OXZ_F32, false},  {16, 345, 3100, OXZ_BF16, OXZ_BF16, false},
        {3, 5764, 32000, OXZ_F32, OXZ_F32, false},   {3, 5763, 32000, OXZ_F32, OXZ_F32, true},
    };
    for (const auto& c : cases) {
        const oxz_head_desc d{c.rows, c.hidden, c.vocab, 0, c.dtype, c.grad, 0, 0};
        oxz_head* h = nullptr;
        uint64_t bytes = 0;
        fake::allocated = 0;
        EXPECT(oxz_head_create(&d, &h) == OXZ_OK);
        EXPECT(oxz_head_alloc(h, &bytes) == OXZ_OK);
        EXPECT(bytes <= fake::allocated && fake::allocated <= bytes + 4096, "%llu reported, %zu taken", (unsigned long long)bytes, fake::allocated);
        // at most: the logits of 16 rows, d_hidden's sums of two blocks an SM of up to 1024 columns each, and small change
        const uint64_t streaming = 64 * (c.vocab + 2 * 148 * std::min<uint64_t>(c.hidden, 1024) + c.hidden) + (1 << 20);
        EXPECT((bytes <= streaming) == c.streams, "%llu rows of %llu over %llu: %llu bytes, streaming alone %llu", (unsigned long long)c.rows, (unsigned long long)c.hidden,
               (unsigned long long)c.vocab, (unsigned long long)bytes, (unsigned long long)streaming);
        for (uint64_t rows = 0; rows <= c.rows; rows++)
            for (uint64_t off : {uint64_t(0), uint64_t(4)}) {
                const oxz_head_batch b{rows, (char*)p + off, 0, p, (const int64_t*)p, nullptr};
                const oxz_head_grads g{p, 0, p, 1.0, 0, 0};
                EXPECT(oxz_head_loss_grads_async(h, &b, (float*)p, nullptr, (float*)p, &g, A) == OXZ_OK, "%s", fake::message.c_str());
            }
        oxz_head_destroy(h);
    }
}

int main(int argc, char** argv) {
    const struct { const char* name; void (*run)(); } tests[] = {
        {"error", an_error_is_reported_once},
        {"broke_off", the_next_call_waits_for_one_that_broke_off},
        {"first", the_first_failure_is_the_one_reported},
        {"handful", a_handful_of_rows_takes_no_workspace_for_tiles},
        {"marks", marks_are_taken_away_after_a_call_that_broke_off},
        {"threads", threads_with_a_handle_each},
    };
    for (const auto& t : tests)
        if (argc < 2 || std::strcmp(argv[1], t.name) == 0) t.run();
    std::printf(failures ? "%d failed\n" : "all passed\n", failures.load());
    return failures != 0;
}
