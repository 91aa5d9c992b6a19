// What the operators around a step's products and a model's filtered sampling launch,
// checked on a machine without a GPU: the library's objects against fake_hip.cpp.
// `step_checks NAME` runs one check.
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

// Pointers that nothing looks behind: no kernel runs.
uint8_t *at(size_t address) { return reinterpret_cast<uint8_t *>(address); }
template <class T>
T *some() {
    return reinterpret_cast<T *>(at(4096));
}

GptConfig shape() {
    GptConfig c;
    c.vocab_size = 64;
    c.context = 64;
    c.width = 128;
    c.heads = 4;
    c.layers = 2;
    c.attention_mesh_depth = 4;
    c.ffn_mesh_depth = 6;
    return c;
}

void draw(Type type, size_t rows, size_t vocab) {
    sample_filtered_noalloc(0, type, at(4096), rows, vocab, vocab, some<float>(), some<int>(), some<float>(), some<float>(),
                            some<float>(), some<uint32_t>(), some<float>(), nullptr);
}
void turn(Type type, size_t batch, size_t count, size_t heads, size_t width, size_t rotary, bool interleaved, bool backward) {
    const Strides s{{int64_t(count * heads * width), int64_t(heads * width), int64_t(width)}};
    rope(0, Rope{width, rotary, interleaved, 1.0f, some<double>()}, type, batch, count, heads, at(4096), s, at(8192), s, 0, nullptr,
         s, nullptr, s, nullptr, nullptr, nullptr, backward, nullptr);
}
void norm(Type type, size_t rows, size_t width, bool codes) {
    if (codes)
        rms_norm_e4m3(0, type, rows, width, at(4096), width, at(4096), width, at(8192), width, at(4096), 1e-5f, at(4096), width,
                      at(4096), width, some<float>(), nullptr);
    else
        rms_norm(0, type, rows, width, at(4096), width, at(4096), width, at(8192), width, at(4096), 1e-5f, at(4096), width,
                 some<float>(), nullptr);
}
void norm_gradient(Type type, size_t rows, size_t width) {
    const size_t room = rms_norm_backward_workspace(rows, width);
    rms_norm_backward(0, type, rows, width, at(4096), width, at(4096), some<float>(), at(4096), width, at(4096), width, at(8192),
                      width, some<float>(), room ? at(16) : nullptr, room, nullptr);
}

const size_t kWidths[] = {1, 130, 512, 1000, 2048, 4100, 8192, 16384};

// Programs that between them launch every kernel of the operators.
std::vector<std::pair<std::string, std::function<void()>>> programs() {
    std::vector<std::pair<std::string, std::function<void()>>> all;
    for (Type type : {Type::F32, Type::F16, Type::BF16}) {
        const std::string name = " of type " + std::to_string(int(type));
        for (size_t vocab : {40, 200, 2000, 20000, 60000, 200000}) all.push_back({"draws" + name, [=] { draw(type, 7, vocab); }});
        for (bool backward : {false, true})
            for (bool interleaved : {false, true}) {
                all.push_back({"turns" + name, [=] { turn(type, 3, 5, 4, 80, 50, interleaved, backward); }});
                all.push_back({"large turns" + name, [=] { turn(type, 16, 8192, 32, 128, 128, interleaved, backward); }});
            }
        for (size_t width : kWidths) {
            all.push_back({"norm" + name, [=] { norm(type, 33, width, false); }});
            all.push_back({"norm to codes" + name, [=] { norm(type, 33, width, true); }});
            all.push_back({"norm gradient" + name, [=] { norm_gradient(type, 33, width); }});
            all.push_back({"large norm gradient" + name, [=] { norm_gradient(type, 3300, width); }});
        }
    }
    all.push_back({"a model", [] {
                       MeshGpt m(0, shape(), 7, 8);
                       m.set_sampling(4, 0.9f, 0.01f);
                       const std::vector<uint32_t> prompts(70 * 20, 1);
                       std::vector<uint32_t> out(8 * 90);
                       m.generate_tokens(prompts.data(), 8, 16, 70, 0.7f, 7, out.data());  // past the context
                       m.prefill(prompts.data(), 70, 20, 0.5f, 7, 40);
                       m.decode(9);
                   }});
    return all;
}

// A launch that the runtime refuses is an error of the call that made it, and the
// same call works afterwards.
void refused_launches() {
    std::set<std::string> every;
    for (const auto &program : programs()) {
        std::set<std::string> kernels;
        fake::on_launch = [&](const fake::Launch &l) {
            kernels.insert(l.kernel);
            expect(double(l.grid.x) * l.block.x < 4294967296.0, "a launch's threads are counted in 32 bits: " + l.kernel);
        };
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
    for (const char *name : {"sample_short_kernel", "sample_bins_kernel", "sample_codes_kernel", "sample_rows_kernel",
                             "sample_append_kernel", "rope_kernel", "norm_kernel", "norm_backward_kernel",
                             "norm_columns_kernel", "norm_rows_kernel", "norm_join_kernel"}) {
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

// The largest calls that are accepted stay inside a launch's limits.
void largest_calls() {
    size_t launches = 0;
    fake::on_launch = [&](const fake::Launch &l) {
        ++launches;
        expect(double(l.grid.x) * l.block.x < 4294967296.0, "a launch's threads are counted in 32 bits: " + l.kernel);
        expect(l.block.x <= 1024, "a workgroup has at most 1024 threads: " + l.kernel);
    };
    const size_t most = (size_t(1) << 22) - 1;
    for (Type type : {Type::F32, Type::F16, Type::BF16}) {
        for (size_t vocab : {1, 1000, 100000, 1 << 20}) draw(type, most, vocab);
        for (size_t width : kWidths) {
            norm(type, most, width, false);
            norm(type, most, width, true);
            norm_gradient(type, most, width);
        }
        for (size_t width : {2, 64, 1024})
            for (bool interleaved : {false, true}) {
                turn(type, 1, (size_t(1) << 24) - 1, 1, width, width, interleaved, false);
                turn(type, 255, 65793, 65536, width, width, interleaved, true);
                turn(type, 3, 5, 65536, width, width, interleaved, true);
                turn(type, 1, 1, 1, width, 0, interleaved, false);
            }
    }
    fake::on_launch = nullptr;
    expect(launches > 0, "calls launch kernels");
}

// Filters that find no memory for their scratch leave the model as it was.
void filters_without_memory() {
    MeshGpt m(0, shape(), 7, 64);
    const std::vector<uint32_t> prompts(64 * 16, 1);
    std::vector<uint32_t> out(64 * 20);
    auto generate = [&] { m.generate_tokens(prompts.data(), 64, 16, 4, 0.7f, 7, out.data()); };
    generate();
    bool through = false;
    fake::on_launch = [&](const fake::Launch &l) { through |= l.kernel.find("sample_append_kernel") != std::string::npos; };
    fake::memory = fake::used;
    expect(status_of([&] { m.set_sampling(3, 1.0f, 0.0f); }) == kOutOfMemory, "no memory for the filters");
    expect(status_of(generate) == 0 && !through, "the model samples as it did");
    fake::memory = size_t(1) << 33;
    expect(status_of([&] { m.set_sampling(3, 1.0f, 0.0f); }) == 0, "the filters are set where there is memory");
    expect(status_of(generate) == 0 && through, "and tokens come through them");
    fake::on_launch = nullptr;
}

// A batch that finds no memory for its filters' scratch is not there: nothing decodes
// from it, and no draw is launched without scratch.
void batch_without_filter_memory() {
    MeshGpt m(0, shape(), 7, 64);
    const std::vector<uint32_t> prompts(64, 1);
    auto begin = [&](float temperature) { m.prefill(prompts.data(), 64, 1, temperature, 7, 20); };
    begin(0.0f);
    m.set_sampling(3, 1.0f, 0.0f);  // a greedy batch needs none
    size_t draws = 0;
    bool scratch = true;
    fake::on_launch = [&](const fake::Launch &l) {
        if (l.kernel.find("sample_rows_kernel") == std::string::npos) return;
        ++draws;
        scratch = scratch && *static_cast<void **>(l.args[0]) != nullptr;
    };
    fake::memory = fake::used;
    expect(status_of([&] { begin(0.7f); }) == kOutOfMemory, "no memory for the filters");
    fake::memory = size_t(1) << 33;
    const bool decoded = status_of([&] { m.decode(1); }) == 0;
    expect(scratch, "no draw is launched without scratch");
    expect(!decoded && m.sequence_length() == 0, "a refused batch does not decode");
    begin(0.7f);
    m.decode(1);
    expect(draws > 0 && scratch, "it is drawn from where there is memory");
    fake::on_launch = nullptr;
}

// A larger batch that is refused for want of memory, wherever it runs out, takes the
// one before with it if that has lost its buffers: nothing decodes from new, empty ones.
void larger_batch_without_memory() {
    const std::vector<uint32_t> prompts(64 * 4, 1);
    bool there = false;
    size_t refused = 0;
    for (size_t room = 0; !there; room += 4096) {
        MeshGpt m(0, shape(), 7, 8);
        m.prefill(prompts.data(), 8, 4, 0.0f, 7, 20);
        std::vector<uint32_t> before(8 * 5), after(8 * 5);
        m.read_tokens(before.data(), 8, 5);
        fake::memory = fake::used + room;
        const int status = status_of([&] { m.prefill(prompts.data(), 64, 4, 0.0f, 7, 20); });
        fake::memory = size_t(1) << 33;
        there = status == 0;
        if (there) continue;
        ++refused;
        expect(status == kOutOfMemory, "a batch without memory is refused");
        if (status_of([&] { m.decode(1); }) != 0) continue;
        expect(m.sequence_length() == 6, "a batch goes on from where it was");
        m.read_tokens(after.data(), 8, 5);
        expect(before == after, "a batch goes on only with its tokens");
    }
    expect(refused > 0, "memory was short");
}

const std::map<std::string, void (*)()> kChecks = {
    {"larger_batch_without_memory", larger_batch_without_memory},
    {"batch_without_filter_memory", batch_without_filter_memory},
    {"refused_launches", refused_launches},
    {"foreign_errors", foreign_errors},
    {"largest_calls", largest_calls},
    {"filters_without_memory", filters_without_memory},
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
