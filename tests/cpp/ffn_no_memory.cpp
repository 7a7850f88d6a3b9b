// Calls of libbvml_ffn.so's entry points while every host allocation fails: each
// returns a status.  (An exception would end the program.)
#include <dlfcn.h>

#include <cstdio>
#include <cstdlib>
#include <new>

#include "bvml_ffn.h"

static bool g_none = false;

void* operator new(std::size_t n) {
    void* p = g_none ? nullptr : std::malloc(n ? n : 1);
    if (!p) throw std::bad_alloc();
    return p;
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }

template <typename F>
static F* symbol(void* lib, const char* name) {
    F* f = reinterpret_cast<F*>(dlsym(lib, name));
    if (!f) {
        std::printf("no %s\n", name);
        std::exit(2);
    }
    return f;
}

int main(int, char** argv) {
    void* lib = dlopen(argv[1], RTLD_NOW);
    if (!lib) {
        std::printf("%s\n", dlerror());
        return 2;
    }
    auto* norm = symbol<decltype(bvml_ffn_add_rms_norm)>(lib, "bvml_ffn_add_rms_norm");
    auto* norm_grad = symbol<decltype(bvml_ffn_add_rms_norm_backward)>(
        lib, "bvml_ffn_add_rms_norm_backward");
    auto* linear = symbol<decltype(bvml_ffn_linear)>(lib, "bvml_ffn_linear");
    auto* gated = symbol<decltype(bvml_ffn_gated)>(lib, "bvml_ffn_gated");
    auto* linear_grad = symbol<decltype(bvml_ffn_linear_backward)>(lib, "bvml_ffn_linear_backward");
    auto* gated_grad = symbol<decltype(bvml_ffn_gated_backward)>(lib, "bvml_ffn_gated_backward");
    auto* plan = symbol<decltype(bvml_ffn_plan)>(lib, "bvml_ffn_plan");
    int status[7];
    g_none = true;  // -1 rows: refused, with a message that cannot be made
    status[0] = norm(nullptr, 0, nullptr, 0, nullptr, -1, 8, 0.0, 0, 0, 0, nullptr, 0, nullptr, 0,
                     nullptr, nullptr, nullptr);
    status[1] = norm_grad(nullptr, 0, nullptr, 0, nullptr, nullptr, nullptr, 0, -1, 8, 0, 0, 0,
                          nullptr, 0, nullptr, nullptr, 0, nullptr);
    status[2] = linear(nullptr, 0, nullptr, 0, nullptr, nullptr, nullptr, nullptr, 0, -1, 8, 8, 2, 2,
                       2, 0, nullptr, 0, nullptr, 0, nullptr, 0, nullptr);
    status[3] = gated(nullptr, 0, nullptr, 0, nullptr, nullptr, nullptr, -1, 8, 8, 2, 2, 2, 0,
                      nullptr, 0, nullptr, 0, nullptr, 0, nullptr);
    status[4] = linear_grad(nullptr, 0, nullptr, 0, nullptr, 0, nullptr, 0, -1, 8, 8, 2, 2, 0,
                            nullptr, 0, nullptr, 0, nullptr, nullptr, 0, nullptr);
    status[5] = gated_grad(nullptr, 0, nullptr, 0, nullptr, 0, nullptr, 0, -1, 8, 8, 2, 2, 0,
                           nullptr, 0, nullptr, 0, nullptr, nullptr, 0, nullptr);
    status[6] = plan(-1, 8, 8, 2, 0, 0, 1, nullptr, nullptr, nullptr, nullptr);
    g_none = false;
    int bad = 0;
    for (int s : status) {
        std::printf("%d ", s);
        bad += s == 0;
    }
    std::printf("\n");
    return bad ? 1 : 0;
}
