// What the device operators and the models' 8-bit cache launch, checked on a
// machine without a GPU: the library's objects against fake_hip.cpp.
// `operator_checks NAME` runs one check.
#include <cstdio>
#include <cstdlib>
#include <functional>
#include <map>
#include <set>
#include <string>
#include <vector>

#include "fake_hip.hpp"
#include "meshgpt_types.hpp"
#include "model.hpp"
#include "operators.hpp"

using namespace meshgpt;

namespace {

void expect(bool ok, const std::string &what) {
    if (ok) return;
    std::fprintf(stderr, "check failed: %s\n", what.c_str());
    std::exit(1);
}

// The status of the Error that f throws, 0 when it returns.
template <class F>
int status_of(F &&f) {
    try {
        f();
    } catch (const Error &e) {
        return e.status;
    }
    return 0;
}

GptConfig shape(size_t W, size_t H, size_t C, size_t L = 2) {
    GptConfig c;
    c.vocab_size = 64;
    c.context = C;
    c.width = W;
    c.heads = H;
    c.layers = L;
    c.attention_mesh_depth = 4;
    c.ffn_mesh_depth = 6;
    return c;
}

void generate(MeshGpt &m, size_t batch, size_t prompt, size_t count) {
    const std::vector<uint32_t> prompts(batch * prompt, 1);
    std::vector<uint32_t> out(batch * (prompt + count));
    m.generate_tokens(prompts.data(), batch, prompt, count, 0.0f, 7, out.data());
}

// Pointers that nothing looks behind: no kernel runs.
uint8_t *at(size_t address) { return reinterpret_cast<uint8_t *>(address); }
template <class T>
T *some() {
    return reinterpret_cast<T *>(at(4096));
}

Kv8 cache(int batch, int heads, int width, int capacity) {
    return Kv8{batch, heads, width, kv8_pad(width), capacity, at(256), at(512), at(768), at(1024)};
}

void attend(const Kv8 &c, Type type, size_t heads, size_t count) {
    const size_t room = kv8_attention_workspace(c, heads, count);
    const Strides s{{int64_t(count * heads * c.width), int64_t(heads * c.width), c.width}};
    kv8_attention(0, c, type, heads, count, at(4096), s, at(8192), s, some<int>(), nullptr, 0.125f, room ? at(16) : nullptr, room,
                  nullptr);
}

void score(Type type, size_t rows, size_t vocab, size_t top) {
    const size_t room = token_logprobs_workspace(rows, vocab, top);
    token_logprobs_noalloc(0, type, at(4096), rows, vocab, vocab, some<uint32_t>(), 1.0f, some<float>(), some<float>(),
                           some<float>(), top, some<uint32_t>(), some<float>(), room ? at(16) : nullptr, room, nullptr);
}

// Programs that between them launch every kernel of the operators.
std::vector<std::pair<std::string, std::function<void()>>> programs() {
    std::vector<std::pair<std::string, std::function<void()>>> all;
    for (Type type : {Type::F32, Type::F16, Type::BF16})
        for (int width : {32, 64, 128, 256}) {
            const std::string name = " of type " + std::to_string(int(type)) + ", width " + std::to_string(width);
            const Strides s{{int64_t(200 * 2 * width), int64_t(2 * width), width}};
            all.push_back({"append" + name, [=] {
                               kv8_append(0, cache(3, 2, width, 256), type, 200, at(4096), s, at(8192), s, some<int>(),
                                          nullptr, nullptr);
                           }});
            all.push_back({"read" + name, [=] {
                               for (int batch : {3, 3000})  // the second's outputs are larger than the caches
                                   kv8_read(0, cache(batch, 2, width, 1024), type, 7, 900, at(4096), s, at(8192), s, nullptr,
                                            nullptr);
                           }});
            all.push_back({"attention of tokens" + name, [=] { attend(cache(2, 2, width, 8192), type, 4, 1); }});
            all.push_back({"attention of prompts" + name, [=] { attend(cache(1, 1, width, 8192), type, 2, 300); }});
        }
    for (Type type : {Type::F32, Type::F16, Type::BF16}) {
        const std::string name = " of type " + std::to_string(int(type));
        all.push_back({"scores" + name, [=] {
                           score(type, 7, 99, 5);
                           score(type, 7, 1000, 5);
                           score(type, 7, 50000, 5);
                       }});
        for (size_t rows : {5, 5000})
            all.push_back({"gradient" + name, [=] {
                               token_logprobs_backward_noalloc(0, type, at(4096), rows, 50000, 50000, some<uint32_t>(), 1.0f,
                                                               some<float>(), some<float>(), some<float>(), some<float>(),
                                                               at(4096), 50000, nullptr);
                           }});
    }
    all.push_back({"scores on host arrays", [] {
                       const std::vector<float> z(3 * 5000, 0.0f);
                       const std::vector<uint32_t> t(3, 1);
                       std::vector<float> lp(3), h(3), best(6);
                       std::vector<uint32_t> ids(6);
                       token_logprobs(0, z.data(), 3, 5000, t.data(), 1.0f, lp.data(), h.data(), 2, ids.data(), best.data());
                   }});
    all.push_back({"a model", [] {
                       MeshGpt m(0, shape(128, 4, 256), 7, 8);
                       m.set_cache(CacheType::E4M3);
                       generate(m, 8, 16, 20);
                       generate(m, 2, 1, 3);
                       const std::vector<uint32_t> prompts(70 * 20, 1);
                       m.prefill(prompts.data(), 70, 20, 0.0f, 7, 40);
                       m.decode(9);  // in slices
                   }});
    return all;
}

// A launch that the runtime refuses is an error of the call that made it, and the
// same call works afterwards.
void refused_launches() {
    std::set<std::string> every;
    for (const auto &program : programs()) {
        std::set<std::string> kernels;
        fake::on_launch = [&](const fake::Launch &l) { kernels.insert(l.kernel); };
        program.second();
        fake::on_launch = nullptr;
        expect(!kernels.empty(), program.first + " launches kernels");
        for (const std::string &k : kernels) {
            fake::refuse = k;
            expect(status_of(program.second) == kDeviceError, program.first + " reports a refused " + k);
            fake::refuse.clear();
        }
        expect(status_of(program.second) == 0, program.first + " runs after refusals");
        every.insert(kernels.begin(), kernels.end());
    }
    for (const char *name : {"kv8_append_kernel", "kv8_read_kernel", "kv8_rows_kernel", "kv8_tiles_kernel", "kv8_join_kernel",
                             "logprob_small_kernel", "logprob_kernel", "logprob_join_kernel", "logprob_backward_kernel"}) {
        bool there = false;
        for (const std::string &k : every) there |= k.find(name) != std::string::npos;
        expect(there, std::string(name) + " is launched");
    }
}

// An error that a program's own HIP calls left on the thread is no error of a call.
void foreign_errors() {
    for (const auto &program : programs()) {
        void *p = nullptr;
        (void)hipMalloc(&p, size_t(1) << 50);
        expect(status_of(program.second) == 0, program.first + " after a foreign error");
    }
}

// Scores on host arrays that find no memory leave none behind.
void scores_without_memory() {
    const std::vector<float> z(3 * 5000, 0.0f);
    const std::vector<uint32_t> t(3, 1);
    std::vector<float> lp(3), h(3);
    const size_t before = fake::used;
    auto call = [&] { token_logprobs(0, z.data(), 3, 5000, t.data(), 1.0f, lp.data(), h.data(), 0, nullptr, nullptr); };
    fake::peak = 0;
    call();
    const size_t need = fake::peak - before;
    for (size_t room : {size_t(0), size_t(100), size_t(60000), size_t(60016), need - 1}) {
        fake::memory = before + room;
        expect(status_of(call) == kOutOfMemory, "no memory for it");
        expect(fake::used == before, "everything is freed");
    }
    fake::memory = before + need;
    expect(status_of(call) == 0 && fake::used == before, "enough for it");
    fake::memory = size_t(1) << 33;
}

// A cache of another type that finds no memory leaves the model with the type that
// it had and no batch.
void cache_without_memory() {
    for (CacheType type : {CacheType::E4M3, CacheType::F32}) {
        const CacheType other = type == CacheType::E4M3 ? CacheType::F32 : CacheType::E4M3;
        MeshGpt m(0, shape(128, 4, 256, type == CacheType::E4M3 ? 2 : 8), 7, 64);
        m.set_cache(other);
        generate(m, 64, 16, 4);
        // Two layers in 8 bits take more than in FP32, eight layers less.
        fake::memory = fake::used;
        expect(status_of([&] { m.set_cache(type); }) == kOutOfMemory, "no memory for the other cache");
        bool rounded = false;
        fake::on_launch = [&](const fake::Launch &l) { rounded |= l.kernel.find("kv8_append_kernel") != std::string::npos; };
        expect(status_of([&] { m.decode(1); }) != 0, "the batch is gone");
        expect(status_of([&] { generate(m, 64, 16, 4); }) == 0, "the model generates in the memory that it had");
        expect(rounded == (other == CacheType::E4M3), "from the cache that it had");
        fake::memory = size_t(1) << 33;
        rounded = false;
        expect(status_of([&] { m.set_cache(type); }) == 0, "the type changes where there is memory");
        generate(m, 64, 16, 4);
        expect(rounded == (type == CacheType::E4M3), "and the model generates from it");
        fake::on_launch = nullptr;
    }
}

// A launch counts its threads in 32 bits: where a batch has more rows to quantise,
// they take several, which between them have every sequence once.
void many_sequences() {
    const size_t batch = (1 << 20) + 3;
    fake::memory = size_t(1) << 40;
    MeshGpt m(0, shape(32, 8, 2, 1), 7, 1);
    m.set_cache(CacheType::E4M3);
    size_t appended = 0, attended = 0;
    const uint8_t *keys = nullptr;
    fake::on_launch = [&](const fake::Launch &l) {
        expect(size_t(l.grid.x) * l.block.x < size_t(1) << 32, "a launch's threads are counted in 32 bits: " + l.kernel);
        if (l.kernel.find("kv8_append_kernel") != std::string::npos) {
            const auto *a = static_cast<const kern::Kv8AppendArgs *>(l.args[0]);
            const int tiles = *static_cast<const int *>(l.args[1]);
            expect(l.grid.x == 2u * unsigned(a->cache.batch * a->cache.heads * tiles), "a workgroup for each tile");
            expect(appended % batch == 0 || a->cache.k == keys, "the sequences follow one another");
            appended += size_t(a->cache.batch);
            keys = a->cache.k + kv8_code_bytes(a->cache);
        }
        if (l.kernel.find("kv8_rows_kernel") != std::string::npos)
            attended += size_t(static_cast<const kern::Kv8AttnArgs *>(l.args[0])->cache.batch);
    };
    generate(m, batch, 1, 2);
    fake::on_launch = nullptr;
    expect(appended == 2 * batch && attended == batch, "every sequence once a token");
    fake::memory = size_t(1) << 33;
}

const std::map<std::string, void (*)()> kChecks = {
    {"refused_launches", refused_launches},
    {"foreign_errors", foreign_errors},
    {"scores_without_memory", scores_without_memory},
    {"cache_without_memory", cache_without_memory},
    {"many_sequences", many_sequences},
};

}  // namespace

int main(int argc, char **argv) {
    const auto check = kChecks.find(argc > 1 ? argv[1] : "");
    if (check == kChecks.end()) {
        for (const auto &c : kChecks) std::puts(c.first.c_str());
        return 2;
    }
    check->second();
    std::puts("ok");
}
