// The entry points of kv4_abi.cu over launchers that fail: each call has to say so, also where the CUDA
// runtime has no error to show. Prints "ok", or the calls that claimed success.
#include <cstdio>
#include <string>

#include "cactus_b200_kv4.h"
#include "kv4/kv4_ops.h"
#include "ops.h"

namespace {
int g_rc = -1;         // what every launcher returns
int g_cuda = 0;        // what the runtime has to show after it
std::string g_message;
}  // namespace

namespace cb {
int abi_fail(int code, const std::string& msg) {
    g_message = msg;
    return code;
}
int abi_check_launch(const char* what) { return g_cuda ? abi_fail(CB_ERR_LAUNCH, std::string(what) + ": of the runtime") : CB_OK; }
namespace kv4 {
int launch_append(const __half*, const __half*, long long, const int*, const int*, const Pages&, int, int, const Geom&, cudaStream_t) { return g_rc; }
int launch_read(const Pages&, const int*, const int*, __half*, __half*, int, int, const Geom&, cudaStream_t) { return g_rc; }
int launch_copy_pages(uint8_t*, long long, long long, long long, int, long long, const int*, const int*, int, cudaStream_t) { return g_rc; }
int launch_compact(const Pages&, const int*, int, long long, const int*, const int*, int, int, const Geom&, cudaStream_t) { return g_rc; }
int launch_attention(const AttnCall&, const Pages&, const Geom&, cudaStream_t) { return g_rc; }
size_t attention_workspace(int, int, int, int, int) { return 16; }
}  // namespace kv4
}  // namespace cb

int main() {
    alignas(64) static uint8_t mem[64];
    uint16_t* h = reinterpret_cast<uint16_t*>(mem);
    int32_t* i = reinterpret_cast<int32_t*>(mem);
    float* f = reinterpret_cast<float*>(mem);
    const size_t page = cactus_cuda_kv4_page_bytes(16, 1, 64, 32);
    bool ok = true;
    auto expect = [&](const char* name, int got, int want, bool message) {
        if (got != want || message != !g_message.empty()) {
            std::printf("%s returned %d, not %d (%s)\n", name, got, want, g_message.c_str());
            ok = false;
        }
        g_message.clear();
    };
    for (int rc : {-1, 0})
        for (int cuda : {0, 1}) {
            g_rc = rc;
            g_cuda = cuda;
            const int want = rc || cuda ? CB_ERR_LAUNCH : CB_OK;
            const bool message = want != CB_OK;
            expect("append", cactus_cuda_kv4_append(h, h, 64, i, i, i, 1, mem, 1, page, 1, 1, 16, 1, 64, 32, nullptr), want, message);
            expect("read", cactus_cuda_kv4_read(mem, 1, page, i, 1, i, i, h, h, 1, 1, 16, 1, 64, 32, nullptr), want, message);
            expect("attention", cactus_cuda_kv4_attention(h, 64, i, i, i, 1, mem, 1, page, h, f, 1, 1, 1, 1, 16, 1, 64, 32, 1.0f, 0, 1, mem, 16, nullptr), want, message);
            expect("copy", cactus_cuda_kv_copy_pages(mem, 1, 16, 16, 1, 0, i, i, 1, nullptr), want, message);
            expect("compact", cactus_cuda_kv4_compact(mem, 1, page, 1, 0, i, i, 1, i, i, 1, 1, 16, 1, 64, 32, nullptr), want, message);
        }
    g_rc = -2;  // too many tiles: the arguments' fault
    g_cuda = 0;
    expect("attention", cactus_cuda_kv4_attention(h, 64, i, i, i, 1, mem, 1, page, h, f, 1, 1, 1, 1, 16, 1, 64, 32, 1.0f, 0, 1, mem, 16, nullptr), CB_ERR_ARG, true);
    if (ok) std::puts("ok");
    return ok ? 0 : 1;
}
