// The entry points of batch_abi.cu and rope_abi.cu over launchers that fail: each call has to say so, also where
// the CUDA runtime has no error to show. Prints "ok", or the calls that claimed success.
#include <cstdio>
#include <string>

#include "batch/batch_ops.h"
#include "cactus_b200_batch.h"
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
namespace batch {
int launch_norm_q8(const NormCall&, cudaStream_t) { return g_rc; }
size_t lora_plan_bytes(long long, long long, long long) { return 16; }
size_t lora_workspace(long long, int) { return 16; }
int launch_lora_plan(const int*, const int*, int, int, int, void*, cudaStream_t) { return g_rc; }
int launch_lora(const LoraCall&, cudaStream_t) { return g_rc; }
int launch_logits(const LogitsCall&, cudaStream_t) { return g_rc; }
}  // namespace batch
namespace kv4 {
int launch_rope_table(float, int, long long, float*, cudaStream_t) { return g_rc; }
int launch_rope_append(const RopeCall&, const Pages&, const Geom&, cudaStream_t) { return g_rc; }
}  // namespace kv4
}  // namespace cb

int main() {
    alignas(64) static uint8_t mem[64], other[64];
    uint16_t *h = reinterpret_cast<uint16_t*>(mem), *o = reinterpret_cast<uint16_t*>(other);
    int32_t* i = reinterpret_cast<int32_t*>(mem);
    uint32_t* u = reinterpret_cast<uint32_t*>(mem);
    float* f = reinterpret_cast<float*>(mem);
    bool ok = true;
    auto expect = [&](const char* name, int got, int want) {
        if (got != want || (want != CB_OK) != !g_message.empty()) {
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
            expect("norm", cactus_cuda_add_rms_norm_q8(h, 8, nullptr, 0, h, nullptr, 0, reinterpret_cast<int8_t*>(mem), f, nullptr, 1, 8, 0.0f, nullptr), want);
            expect("plan", cactus_cuda_lora_plan(i, i, 1, 1, 1, mem, 16, nullptr), want);
            expect("lora", cactus_cuda_lora_f16(h, 8, h, h, nullptr, nullptr, nullptr, 0, o, 8, mem, 16, 1, 1, 1, 8, 8, 8, mem, 16, nullptr), want);
            expect("logits", cactus_cuda_logits_process_f16(h, 8, h, 8, 1, 8, f, u, i, nullptr, 1, u, f, i, 1, u, 1, 1, nullptr, nullptr), want);
            expect("table", cactus_cuda_rope_table(1e4f, 16, 1, f, nullptr), want);
            expect("rope", cactus_cuda_kv4_rope_append(h, 64, o, 64, h, h, 64, f, 1, 64, nullptr, nullptr, 0.0f, i, i, i, 1, mem, 1, 16 * (64 + 16), 1, 1, 1, 16, 1, 64, 32, nullptr), want);
        }
    if (ok) std::puts("ok");
    return ok ? 0 : 1;
}
