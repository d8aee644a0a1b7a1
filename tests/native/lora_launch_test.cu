// How lora.cu and lora_tc.cu launch the adapters' kernels, without a GPU: the runtime's calls are wrapped (by the linker)
// and recorded. The second product's kernel starts while the first one's runs and reads the plan and the base before it
// waits for it, so the first one must start only when all that was launched before it is done, also where the caller's
// thread has programmatic launches switched on. Prints "ok", or what was launched otherwise.
#include <cstdio>
#include <vector>

#include "batch/batch_ops.h"
#include "common.cuh"

namespace cb {
__device__ unsigned g_dev_error = 0;
bool& pdl_flag() {
    static bool f = false;
    return f;
}
}  // namespace cb

namespace {
struct Launch {
    bool programmatic;
    unsigned cluster;
};
std::vector<Launch> g_launches;
unsigned g_word;
}  // namespace

extern "C" {
cudaError_t __wrap_cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void*, void**) {
    Launch l = {false, 1};
    for (unsigned i = 0; i < c->numAttrs; ++i) {
        if (c->attrs[i].id == cudaLaunchAttributeProgrammaticStreamSerialization)
            l.programmatic = c->attrs[i].val.programmaticStreamSerializationAllowed != 0;
        if (c->attrs[i].id == cudaLaunchAttributeClusterDimension) l.cluster = c->attrs[i].val.clusterDim.x;
    }
    g_launches.push_back(l);
    return cudaSuccess;
}
cudaError_t __wrap_cudaGetDevice(int* d) {
    *d = 0;
    return cudaSuccess;
}
cudaError_t __wrap_cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t __wrap_cudaGetSymbolAddress(void** p, const void*) {
    *p = &g_word;
    return cudaSuccess;
}
}

int main() {
    bool ok = true;
    alignas(16) static uint8_t mem[64];  // nothing of it is read
    struct Case {
        const char* name;
        int seqs, tokens, max_rank, k, n, launches;
    };
    const Case cases[] = {{"a cluster a tile", 4, 4, 16, 64, 64, 1},
                          {"both products by lora.cu", 1, 100, 16, 64, 64, 2},
                          {"the second one by lora_tc.cu", 1, 520, 32, 128, 8192, 2},
                          {"both by lora_tc.cu, 64", 1, 512, 64, 2048, 2048, 2},
                          {"both by lora_tc.cu, 128", 1, 512, 128, 2048, 2048, 2}};
    for (const Case& at : cases)
        for (bool outer : {false, true}) {
            cb::pdl_scope scope(outer);
            cb::batch::LoraCall c = {};
            __half* p = reinterpret_cast<__half*>(mem);
            c.x = c.a = c.b = c.base = p;
            c.out = p;
            c.x_stride = at.k;
            c.base_stride = c.out_stride = at.n;
            c.plan = reinterpret_cast<int*>(mem);
            c.num_seqs = at.seqs, c.num_tokens = at.tokens, c.num_adapters = 4, c.max_rank = at.max_rank, c.k = at.k, c.n = at.n;
            c.ws = reinterpret_cast<float*>(mem);
            g_launches.clear();
            const int rc = cb::batch::launch_lora(c, nullptr);
            const bool count = rc == 0 && (int)g_launches.size() == at.launches;
            const bool first = count && !g_launches[0].programmatic && (g_launches[0].cluster > 1) == (at.launches == 1);
            const bool second = count && (at.launches == 1 || g_launches[1].programmatic);
            if (!count || !first || !second || cb::pdl_flag() != outer) {
                std::printf("%s, %s: rc %d, %zu launches, first %s, second %s\n", at.name, outer ? "programmatic" : "plain", rc,
                            g_launches.size(), first ? "as it should" : "not", second ? "as it should" : "not");
                ok = false;
            }
        }
    if (ok) std::puts("ok");
    return ok ? 0 : 1;
}
