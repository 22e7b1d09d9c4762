// Tests of the C++ host layer over include/ext (glm53f-afd_amd/host/lin.hpp, spec.hpp, and Gemm::fused of gemm.hpp).
// `--cpu`: what the wrappers reject, without touching a GPU. `--gpu`: a speculative round through them - a fused projection,
// a prompt, a verify window, probabilities, the verification and the commit by its counts on the device - against the
// same arithmetic in double on the host.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "gemm.hpp"
#include "kda_ref.h"   // the oracle's bf16 conversions and generator: test infrastructure
#include "lin.hpp"
#include "spec.hpp"

using namespace glm53f_lin;
using glm53f_forward::Bf16Mat;
using glm53f_forward::Epilogue;
using glm53f_forward::Gemm;
using glm53f_kda::device_count;

static int failures = 0;
#define EXPECT(cond)                                                          \
    do {                                                                      \
        if (!(cond)) {                                                        \
            std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond);       \
            ++failures;                                                       \
        }                                                                     \
    } while (0)
#define EXPECT_OK(expr)                                                       \
    do {                                                                      \
        Error e_ = (expr);                                                    \
        if (!e_) {                                                            \
            std::printf("FAIL %s:%d: %s -> %s\n", __FILE__, __LINE__, #expr, e_.what.c_str()); \
            ++failures;                                                       \
        }                                                                     \
    } while (0)
#define EXPECT_INVALID(expr)                                                  \
    do {                                                                      \
        Error e_ = (expr);                                                    \
        if (e_.kind != Error::Invalid) {                                      \
            std::printf("FAIL %s:%d: expected Invalid from %s, got kind %d (%s)\n", __FILE__, __LINE__, #expr, (int)e_.kind, e_.what.c_str()); \
            ++failures;                                                       \
        }                                                                     \
    } while (0)

static Buf fake(size_t bytes, uintptr_t at = 0x100000) { return Buf(reinterpret_cast<void*>(at), bytes); }

static void cpu_tests() {
    const Shape s{4, 2, 128, 64};
    EXPECT_OK(s.check());
    EXPECT(s.state_len() == 4u * 64 * 128 && s.qk_width() == 256 && s.v_width() == 256);
    EXPECT_INVALID((Shape{4, 3, 128, 128}.check()));
    EXPECT_INVALID((Shape{0, 1, 128, 128}.check()));
    EXPECT_INVALID((Shape{4, 4, 96, 128}.check()));
    EXPECT(Workspace::bytes_for(s, 1, 64) == 0 && Workspace::bytes_for(s, 1, 1 << 20) > 0 && Workspace::bytes_for(s, 0, 64) == -1);
    for (size_t b = 1; b < 300; b += 7)
        for (size_t r = 1; r < 100000; r += 1 + r / 3) EXPECT(Workspace::bytes_for(s, b, r) <= (int64_t)Workspace::bound(s, b, r));

    const size_t n = s.state_len();
    BatchMeta meta(3);
    EXPECT_OK(meta.set({{2, 0, n}, {0, 0, 0}, {5, 0, 2 * n}}));
    Attention a;
    a.shape = s;
    a.q = RowView(fake(7 * 1024 * 2), 0, 1024);
    a.k = RowView(fake(7 * 1024 * 2), 256, 1024);
    a.v = RowView(fake(7 * 1024 * 2), 512, 1024);
    a.log_decay = fake(16);
    a.state = fake(3 * n * 4);
    a.state_out = StateOut::in_place();
    a.out = RowView::dense(fake(7 * 256 * 2), 256);
    void* so = nullptr;
    EXPECT_OK(a.check(meta, StateType::F32, &so));
    EXPECT(so == a.state.p);
    { Attention b = a; b.state_out = StateOut::skip(); EXPECT_OK(b.check(meta, StateType::F32, &so)); EXPECT(so == nullptr); }
    { Attention b = a; b.state = fake(3 * n * 2); EXPECT_OK(b.check(meta, StateType::Bf16, &so)); EXPECT_INVALID(b.check(meta, StateType::F32, &so)); }
    { Attention b = a; b.q = RowView(fake(6 * 1024 * 2), 0, 1024); EXPECT_INVALID(b.check(meta, StateType::F32, &so)); }
    { Attention b = a; b.out.stride = 255; EXPECT_INVALID(b.check(meta, StateType::F32, &so)); }
    { Attention b = a; b.log_decay = fake(12); EXPECT_INVALID(b.check(meta, StateType::F32, &so)); }
    { Attention b = a; b.state_out = StateOut::to(a.state); EXPECT_INVALID(b.check(meta, StateType::F32, &so)); }
    { Attention b = a; b.state_out = StateOut::to(fake(n * 4, 0x9000000)); EXPECT_INVALID(b.check(meta, StateType::F32, &so)); }
    { BatchMeta m(3); EXPECT_OK(m.set({{2, 0, 0}, {1, 0, n / 2}})); EXPECT_INVALID(a.check(m, StateType::F32, &so)); }   // states overlap
    { BatchMeta m(3); EXPECT_OK(m.set({{2, 0, 4}})); EXPECT_INVALID(a.check(m, StateType::F32, &so)); }                  // offset of 4
    EXPECT_INVALID(a.launch_chain(meta, StateType::F32, Stream::null()));   // no device arrays
    { BatchMeta m(1); EXPECT_OK(m.set({{200000, 0, 0}})); Attention b = a;
      b.q = b.k = b.v = RowView(fake(size_t(200000) * 2048), 0, 1024); b.out = RowView::dense(fake(size_t(200000) * 512), 256);
      EXPECT_INVALID(b.launch_prefill(m, StateType::F32, nullptr, Stream::null())); }                                    // workspace missing

    auto commit = [&](size_t layers, size_t rl, size_t sl, size_t decays, size_t state) {
        return advance_batch(s, layers, meta, nullptr, a.k, a.v, rl, fake(decays * 4), fake(state * 4), sl, StateType::F32, Stream::null(), true);
    };
    EXPECT_OK(commit(1, 0, 0, 4, 3 * n));
    EXPECT_INVALID(commit(0, 0, 0, 4, 3 * n));
    EXPECT_INVALID(commit(2, 0, 2 * n, 8, 6 * n));      // layers' states overlap
    EXPECT_OK(commit(2, 0, 3 * n, 8, 6 * n));
    EXPECT_INVALID(commit(2, 0, 3 * n, 4, 6 * n));      // decays of one layer
    EXPECT_INVALID(commit(2, 7 * 1024, 3 * n, 8, 6 * n));   // rows of one layer
    EXPECT_INVALID(commit(1, 0, 0, 4, 2 * n));

    glm53f_spec::Workspace none;
    glm53f_spec::Probabilities p;
    p.rows = 4; p.vocab = 100;
    p.logits = RowView::dense(fake(400 * 2), 100);
    p.probs = RowView::dense(fake(400 * 4), 100);
    EXPECT_INVALID(p.check(none));                      // no workspace
    EXPECT(glm53f_spec::Workspace::bytes_for(4, 3, 100) > 0 && glm53f_spec::Workspace::bytes_for(70000, 1, 100) == -1);
    p.logits.stride = 99;
    EXPECT_INVALID(p.check(none));
    glm53f_spec::Verification v;
    v.vocab = 100;
    v.tokens = v.uniform = fake(7 * 4);
    v.keep = v.next = fake(12);
    v.target = RowView::dense(fake(700 * 4), 100);
    EXPECT_INVALID(v.check(meta, none));                // no workspace
    v.tokens = fake(6 * 4);
    EXPECT_INVALID(v.check(meta, none));

    const uint16_t* wp = reinterpret_cast<const uint16_t*>(uintptr_t(0x10000));
    Epilogue e;
    e.act = 9;
    EXPECT_INVALID(Gemm::fused(wp, 64, 0, Bf16Mat{wp, 32, 64, 64}, 4, e, const_cast<uint16_t*>(wp), 32, 0, false, Stream::null()));
    e.act = GLM53F_ACT_SILU;
    EXPECT_OK(Gemm::fused(nullptr, 64, 0, Bf16Mat{wp, 32, 64, 64}, 0, e, nullptr, 32, 0, false, Stream::null()));   // no rows
}

static float widen(uint16_t b) { uint32_t u = (uint32_t)b << 16; float f; std::memcpy(&f, &u, 4); return f; }
static uint16_t narrow(float f) {
    uint32_t u; std::memcpy(&u, &f, 4);
    return (uint16_t)((u + 0x7fff + ((u >> 16) & 1)) >> 16);
}

struct Lcg {
    uint64_t s;
    float next() { s = s * 6364136223846793005ull + 1442695040888963407ull; return (float)((s >> 40) / 8388608.0 - 1.0); }
};

static void gpu_tests() {
    Stream stream = Stream::null();
    Lcg rng{7};
    const Shape s{4, 2, 64, 128};
    const size_t n = s.state_len(), width = 2 * s.qk_width() + s.v_width(), k_in = 96, vocab = 300;
    const std::vector<size_t> lens = {4, 1, 7};
    const size_t total = 12;
    auto bf16 = [&](size_t count, float scale) { std::vector<uint16_t> x(count); for (auto& v : x) v = narrow(rng.next() * scale); return x; };
    // the projection of the hidden rows into q | k | v, with a bias
    const auto x = bf16(total * k_in, 1.0f), w = bf16(width * k_in, 0.2f), bias = bf16(width, 0.3f);
    DeviceBuffer dx, dw, db, rows, state, decay, out;
    EXPECT_OK(DeviceBuffer::from_slice(x, &dx));
    EXPECT_OK(DeviceBuffer::from_slice(w, &dw));
    EXPECT_OK(DeviceBuffer::from_slice(bias, &db));
    EXPECT_OK(DeviceBuffer::alloc(total * width * 2, &rows));
    Epilogue e;
    e.bias = db.ptr<uint16_t>();
    EXPECT_OK(Gemm::fused(dx.ptr<uint16_t>(), k_in, 0, Bf16Mat{dw.ptr<uint16_t>(), width, k_in, k_in}, total, e, rows.ptr<uint16_t>(), width, 0,
                          false, stream));
    std::vector<uint16_t> qkv;
    EXPECT_OK(rows.to_vec(&qkv));
    for (size_t r = 0; r < total; ++r)
        for (size_t o = 0; o < width; ++o) {
            double y = widen(bias[o]), a = std::fabs(y);
            for (size_t i = 0; i < k_in; ++i) { const double p = (double)widen(x[r * k_in + i]) * widen(w[o * k_in + i]); y += p; a += std::fabs(p); }
            EXPECT(std::fabs(widen(qkv[r * width + o]) - y) <= std::fabs(y) / 256 + (k_in + 1) * a / 16777216);
        }
    // a verify window of every request over its state
    std::vector<float> state0(3 * n), g(s.heads);
    for (auto& v : state0) v = rng.next() * 0.5f;
    for (size_t h = 0; h < s.heads; ++h) g[h] = -0.1f * (float)(h + 1);
    EXPECT_OK(DeviceBuffer::from_slice(state0, &state));
    EXPECT_OK(DeviceBuffer::from_slice(g, &decay));
    EXPECT_OK(DeviceBuffer::zeroed(total * s.v_width() * 2, &out));
    BatchMeta meta(0);
    EXPECT_OK(BatchMeta::create(3, &meta));
    const std::vector<size_t> slot = {2 * n, 0, n};
    EXPECT_OK(meta.set({{lens[0], 0, slot[0]}, {lens[1], 0, slot[1]}, {lens[2], 0, slot[2]}}));
    Attention at;
    at.shape = s;
    at.q = RowView(rows, 0, width);
    at.k = RowView(rows, s.qk_width(), width);
    at.v = RowView(rows, 2 * s.qk_width(), width);
    at.log_decay = decay;
    at.scale = 0.125f;
    at.state = state;
    at.state_out = StateOut::skip();
    at.out = RowView::dense(out, s.v_width());
    Workspace ws;
    EXPECT_OK(Workspace::create(s, 3, 7, &ws));
    EXPECT_OK(at.launch_prefill(meta, StateType::F32, &ws, stream));
    std::vector<uint16_t> o_prefill, o_chain;
    EXPECT_OK(out.to_vec(&o_prefill));
    EXPECT_OK(at.launch_chain(meta, StateType::F32, stream));
    EXPECT_OK(out.to_vec(&o_chain));
    // logits of the windows, their probabilities, and the verification: the tokens are the most probable ones of the first
    // request's rows, so that it keeps them all but the last (another token)
    std::vector<float> logits(total * vocab), uniform(total, 0.3f);
    for (auto& v : logits) v = rng.next() * 3.0f;
    std::vector<int32_t> tokens(total, 0);
    for (size_t r = 1; r < 3; ++r) { tokens[r] = (int32_t)(10 * r); logits[(r - 1) * vocab + 10 * r] = 30.0f; }
    tokens[3] = 5; logits[2 * vocab + 5] = -40.0f;
    for (size_t r = 6; r < 12; ++r) { tokens[r] = (int32_t)(7 * r); logits[(r - 1) * vocab + 7 * r] = 30.0f; }
    DeviceBuffer dl, dt, du, keep, next;
    EXPECT_OK(DeviceBuffer::from_slice(logits, &dl));
    EXPECT_OK(DeviceBuffer::from_slice(tokens, &dt));
    EXPECT_OK(DeviceBuffer::from_slice(uniform, &du));
    EXPECT_OK(DeviceBuffer::zeroed(12, &keep));
    EXPECT_OK(DeviceBuffer::zeroed(12, &next));
    glm53f_spec::Workspace sw;
    EXPECT_OK(glm53f_spec::Workspace::create(total, 3, vocab, &sw));
    glm53f_spec::Probabilities p;
    p.rows = total; p.vocab = vocab; p.logits_f32 = true;
    p.logits = p.probs = RowView::dense(dl, vocab);     // in place
    EXPECT_OK(p.launch(sw, stream));
    glm53f_spec::Verification v;
    v.vocab = vocab;
    v.tokens = dt; v.uniform = du; v.keep = keep; v.next = next;
    v.target = RowView::dense(dl, vocab);
    EXPECT_OK(v.launch(meta, sw, stream));
    // the commit by the counts on the device
    EXPECT_OK(advance_batch(s, 1, meta, keep.ptr<int32_t>(), at.k, at.v, 0, decay, state, 0, StateType::F32, stream));
    std::vector<int32_t> kept, token;
    std::vector<float> probs, state1;
    EXPECT_OK(keep.to_vec(&kept));
    EXPECT_OK(next.to_vec(&token));
    EXPECT_OK(dl.to_vec(&probs));
    EXPECT_OK(state.to_vec(&state1));
    EXPECT(kept[0] == 3 && kept[1] == 1 && kept[2] == 7);
    for (size_t r = 0; r < total; ++r) {
        double sum = 0, top = -1e30;
        for (size_t t = 0; t < vocab; ++t) top = std::max(top, (double)logits[r * vocab + t]);
        for (size_t t = 0; t < vocab; ++t) sum += std::exp(logits[r * vocab + t] - top);
        for (size_t t = 0; t < vocab; ++t) {
            const double want = std::exp(logits[r * vocab + t] - top) / sum;
            EXPECT(std::fabs(probs[r * vocab + t] - want) <= want * 3e-5 + 1e-37);
        }
    }
    const size_t row_of[3] = {2, 4, 11};                // the last kept row of each window
    for (size_t b = 0; b < 3; ++b) {
        double all = 0, run = 0;
        int want = -1;
        auto weight = [&](size_t t) { return b == 0 && t == 5 ? 0.0 : (double)probs[row_of[b] * vocab + t]; };   // the rejected draft is left out
        for (size_t t = 0; t < vocab; ++t) all += weight(t);
        for (size_t t = 0; t < vocab && want < 0; ++t) { run += weight(t); if (run > (double)0.3f * all) want = (int)t; }
        EXPECT(token[b] == want);
    }
    // outputs and states against the recurrence in double
    const size_t first[3] = {0, 4, 5};
    for (size_t b = 0; b < 3; ++b)
        for (size_t h = 0; h < s.heads; ++h) {
            std::vector<double> st(s.value_dim * s.key_dim), ab(st.size());
            for (size_t i = 0; i < st.size(); ++i) { st[i] = state0[slot[b] + h * st.size() + i]; ab[i] = std::fabs(st[i]); }
            for (size_t t = 0; t < lens[b]; ++t) {
                const uint16_t* row = &qkv[(first[b] + t) * width];
                const uint16_t *q = row + (h / 2) * s.key_dim, *k = row + s.qk_width() + (h / 2) * s.key_dim, *vv = row + 2 * s.qk_width() + h * s.value_dim;
                for (size_t d = 0; d < s.value_dim; ++d) {
                    double o = 0, oa = 0;
                    for (size_t i = 0; i < s.key_dim; ++i) {
                        const double add = (double)widen(vv[d]) * widen(k[i]), f = std::exp((double)g[h]);
                        double& z = st[d * s.key_dim + i];
                        double& za = ab[d * s.key_dim + i];
                        z = f * z + add, za = f * za + std::fabs(add);
                        o += 0.125 * z * widen(q[i]), oa += 0.125 * za * std::fabs(widen(q[i]));
                    }
                    const size_t at_o = (first[b] + t) * s.v_width() + h * s.value_dim + d;
                    const double tol = std::fabs(o) / 256 + oa / 65536;
                    EXPECT(std::fabs(widen(o_prefill[at_o]) - o) <= tol && std::fabs(widen(o_chain[at_o]) - o) <= tol);
                }
                if ((int)t + 1 == kept[b])
                    for (size_t i = 0; i < st.size(); ++i)
                        EXPECT(std::fabs(state1[slot[b] + h * st.size() + i] - st[i]) <= (lens[b] + 16) * ab[i] / 16777216);
            }
        }
}

int main(int argc, char** argv) {
    const std::string mode = argc > 1 ? argv[1] : "--cpu";
    cpu_tests();
    if (mode == "--gpu") {
        if (device_count() == 0) { std::printf("no GPU\n"); return 2; }
        gpu_tests();
    }
    if (failures) { std::printf("%d failures\n", failures); return 1; }
    std::printf("ext host tests passed (%s)\n", mode.c_str());
    return 0;
}
