// Which states the linear attention's wrappers (glm53f-afd_amd/host/lin.hpp) take together: argument checks on made-up
// addresses, no GPU.
#include <cstdio>
#include <string>
#include <vector>

#include "lin.hpp"

using namespace glm53f_lin;

static int failures = 0;
#define EXPECT(cond)                                                    \
    do {                                                                \
        if (!(cond)) {                                                  \
            std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            ++failures;                                                 \
        }                                                               \
    } while (0)

static Buf fake(size_t bytes, uintptr_t at) { return Buf(reinterpret_cast<void*>(at), bytes); }

static const Shape kShape{4, 2, 128, 64};
static const uintptr_t kPool = 0x10000000;

static Attention attention(size_t rows) {
    Attention a;
    a.shape = kShape;
    a.q = RowView(fake(rows * 1024 * 2, 0x100000), 0, 1024);
    a.k = RowView(fake(rows * 1024 * 2, 0x100000), 256, 1024);
    a.v = RowView(fake(rows * 1024 * 2, 0x100000), 512, 1024);
    a.log_decay = fake(16, 0x80000);
    a.state = fake(6 * kShape.state_len() * 4, kPool);
    a.out = RowView::dense(fake(rows * 256 * 2, 0x800000), 256);
    return a;
}

static Error::Kind kind(const Attention& a, const BatchMeta& meta, StateType st = StateType::F32) {
    void* so = nullptr;
    return a.check(meta, st, &so).kind;
}

// Several windows behind one state are a call that only reads them; where states are written each request has its own.
static void windows_of_one_state() {
    const size_t n = kShape.state_len();
    BatchMeta meta(3);
    EXPECT(meta.set({{2, 0, n}, {1, 0, n}, {4, 0, 0}}).is_ok());
    Attention a = attention(7);
    a.state_out = StateOut::skip();
    EXPECT(kind(a, meta) == Error::Ok && kind(a, meta, StateType::Bf16) == Error::Ok);
    a.state_out = StateOut::in_place();
    EXPECT(kind(a, meta) == Error::Invalid);
    a.state_out = StateOut::to(fake(3 * n * 4, 2 * kPool));
    EXPECT(kind(a, meta) == Error::Invalid);
    a.state_out = StateOut::skip();
    EXPECT(meta.set({{2, 0, 6 * n}}).is_ok());
    EXPECT(kind(a, meta) == Error::Invalid);            // outside the pool
}

// States written to another buffer lie apart from every state that is read, also where the buffers are parts of one allocation.
static void states_written_elsewhere() {
    const size_t n = kShape.state_len(), bytes = n * 4;
    BatchMeta meta(3);
    EXPECT(meta.set({{2, 0, n}, {1, 0, 3 * n}, {0, 0, 5 * n}}).is_ok());
    Attention a = attention(3);
    auto to = [&](uintptr_t at, size_t size) { a.state_out = StateOut::to(fake(size, at)); return kind(a, meta); };
    EXPECT(to(2 * kPool, 6 * bytes) == Error::Ok);
    EXPECT(to(kPool + 6 * bytes, 6 * bytes) == Error::Ok && to(kPool - 6 * bytes, 6 * bytes) == Error::Ok);
    EXPECT(to(kPool + bytes, 6 * bytes) == Error::Ok && to(kPool - bytes, 6 * bytes) == Error::Ok);   // the slots between
    EXPECT(to(kPool + 2 * bytes, 6 * bytes) == Error::Invalid);      // the next request's
    EXPECT(to(kPool - 4 * bytes, 6 * bytes) == Error::Invalid);
    EXPECT(to(kPool + 16, 6 * bytes) == Error::Invalid && to(kPool - 16, 6 * bytes) == Error::Invalid);   // its own in part
    EXPECT(to(kPool + bytes + 16, 6 * bytes) == Error::Invalid && to(kPool + bytes - 16, 6 * bytes) == Error::Invalid);
    EXPECT(to(kPool, 6 * bytes) == Error::Invalid);                  // InPlace
    a.state = fake(6 * n * 2, kPool);
    a.state_out = StateOut::to(fake(6 * n * 2, kPool + n * 2));
    EXPECT(kind(a, meta, StateType::Bf16) == Error::Ok);
    a.state_out = StateOut::to(fake(6 * n * 2, kPool + 2 * n * 2));
    EXPECT(kind(a, meta, StateType::Bf16) == Error::Invalid);
}

int main() {
    windows_of_one_state();
    states_written_elsewhere();
    if (failures) { std::printf("%d failures\n", failures); return 1; }
    std::printf("state checks passed\n");
    return 0;
}
