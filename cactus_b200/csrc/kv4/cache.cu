// The 4-bit paged KV cache as a handle: a pool for all layers, the sequences' pages (page_map.h) and
// the current batch's metadata in device memory. The device work is the kernel entry points'.
#include <algorithm>
#include <cstring>
#include <memory>
#include <new>
#include <string>
#include <vector>

#include "../../../include/cactus_b200_kv4.h"
#include "../ops.h"
#include "page_map.h"

namespace {

using cb::abi_fail;
using cb::kv4::PageMap;

struct CudaError : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void cu(cudaError_t e, const char* what) {
    if (e != cudaSuccess) throw CudaError(std::string(what) + ": " + cudaGetErrorString(e));
}
// the device of a cache for the length of a call
struct OnDevice {
    int prev = -1;
    explicit OnDevice(int device) {
        cu(cudaGetDevice(&prev), "cudaGetDevice");
        cu(cudaSetDevice(device), "cudaSetDevice");
    }
    ~OnDevice() { cudaSetDevice(prev); }
};

// Host integers on their way to the device: pinned blocks used in turn, each free again when the copy
// from it is done.
class Staging {
public:
    void init(size_t ints) {
        ints_ = ints;
        for (auto& s : slots_) {
            cu(cudaMallocHost(&s.host, ints * 4), "cudaMallocHost");
            cu(cudaEventCreateWithFlags(&s.done, cudaEventDisableTiming), "cudaEventCreate");
        }
    }
    ~Staging() {
        for (auto& s : slots_) {
            if (s.done) cudaEventDestroy(s.done);
            if (s.host) cudaFreeHost(s.host);
        }
    }
    void send(const std::vector<int>& v, int* device, cudaStream_t st) {
        if (v.size() > ints_) throw std::length_error("batch metadata too large");
        Slot& s = slots_[next_];
        next_ = (next_ + 1) % kSlots;
        cu(cudaEventSynchronize(s.done), "cudaEventSynchronize");
        std::memcpy(s.host, v.data(), v.size() * 4);
        cu(cudaMemcpyAsync(device, s.host, v.size() * 4, cudaMemcpyHostToDevice, st), "cudaMemcpyAsync");
        cu(cudaEventRecord(s.done, st), "cudaEventRecord");
    }

private:
    static constexpr int kSlots = 4;
    struct Slot {
        int* host = nullptr;
        cudaEvent_t done = nullptr;
    };
    Slot slots_[kSlots];
    size_t ints_ = 0;
    int next_ = 0;
};

struct Cache {
    size_t layers, hkv, d, g, page, num_pages, max_seqs, max_pages, max_tokens, hq, page_bytes;
    int device = 0;
    std::unique_ptr<PageMap> map;
    Staging staging;
    uint8_t* pool = nullptr;  // [layer][page][page_bytes]
    uint8_t* ws = nullptr;
    size_t ws_bytes = 0;
    int* meta = nullptr;      // the batch: offsets [max_seqs + 1] | lengths [max_seqs] | table [sequences][batch_pages]
    int* lists = nullptr;     // copies, or a compaction's tables and rows
    size_t list_ints = 0;
    size_t batch = 0, batch_tokens = 0, batch_longest = 0, batch_pages = 0;  // pages: of the longest, the table's width

    ~Cache() {
        int prev = -1;
        if (cudaGetDevice(&prev) == cudaSuccess) cudaSetDevice(device);
        for (void* p : {(void*)pool, (void*)ws, (void*)meta, (void*)lists})
            if (p) cudaFree(p);
        if (prev >= 0) cudaSetDevice(prev);
    }
    const int* offsets() const { return meta; }
    const int* lens() const { return meta + max_seqs + 1; }
    const int* table() const { return meta + 2 * max_seqs + 1; }
    uint8_t* layer_pool(size_t l) const { return pool + l * num_pages * page_bytes; }
};

std::vector<int> ints(const int32_t* p, size_t n) { return std::vector<int>(p, p + n); }

// every entry point: no exception leaves, the device is the cache's, failures leave a message
template <typename F>
int guarded(cactus_kv4_t h, const char* name, F f) {
    if (!h) return abi_fail(CB_ERR_ARG, std::string(name) + ": null cache");
    try {
        Cache& c = *static_cast<Cache*>(h);
        OnDevice on(c.device);
        return f(c);
    } catch (const CudaError& e) {
        return abi_fail(CB_ERR_LAUNCH, std::string(name) + ": " + e.what());
    } catch (const std::exception& e) {
        return abi_fail(CB_ERR_ARG, std::string(name) + ": " + e.what());
    } catch (...) {
        return abi_fail(CB_ERR_ARG, std::string(name) + ": unknown error");
    }
}
void require(bool ok, const char* why) {
    if (!ok) throw std::invalid_argument(why);
}
// The stream of a call. A captured one would be wrong when it is replayed after the next begin: the batch's
// counts and the table's width are arguments of the launches, and page lists pass through host memory.
cudaStream_t stream_of(void* stream) {
    cudaStreamCaptureStatus status;
    cu(cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &status), "cudaStreamIsCapturing");
    require(status == cudaStreamCaptureStatusNone, "a cache's calls cannot be captured (its kernel entry points can)");
    return static_cast<cudaStream_t>(stream);
}

}  // namespace

extern "C" {

CB_API cactus_kv4_t cactus_kv4_create(size_t num_layers, size_t num_q_heads, size_t num_kv_heads, size_t head_dim,
                                      size_t group_size, size_t page_size, size_t num_pages, size_t max_seqs,
                                      size_t max_context, size_t max_tokens, int device) {
    try {
        auto c = std::make_unique<Cache>();
        c->layers = num_layers;
        c->hq = num_q_heads;
        c->hkv = num_kv_heads;
        c->d = head_dim;
        c->g = group_size;
        c->page = page_size;
        c->num_pages = num_pages;
        c->max_seqs = max_seqs;
        c->max_tokens = max_tokens;
        c->device = device;
        c->page_bytes = cactus_cuda_kv4_page_bytes(page_size, num_kv_heads, head_dim, group_size);
        require(c->page_bytes != 0, "unsupported page_size, num_kv_heads, head_dim or group_size");
        require(num_layers >= 1 && num_layers <= 65535, "num_layers must be 1 to 65535");
        require(num_q_heads >= 1 && num_q_heads % num_kv_heads == 0 && num_q_heads <= 65536,
                "num_q_heads must be a multiple of num_kv_heads");
        require(num_pages >= 1 && num_pages < (size_t(1) << 30), "num_pages must be 1 to 2^30");
        require(num_layers <= (size_t(1) << 62) / c->page_bytes / num_pages, "the pool would have more than 2^62 bytes");
        require(max_seqs >= 1 && max_seqs <= (size_t(1) << 20), "max_seqs must be 1 to 2^20");
        require(max_context >= 1 && max_context <= (size_t(1) << 30), "max_context must be 1 to 2^30");
        require(max_tokens >= 1 && max_tokens <= (size_t(1) << 30), "max_tokens must be 1 to 2^30");
        c->max_pages = (max_context + page_size - 1) / page_size;
        require(c->max_pages * max_seqs < (size_t(1) << 30), "max_seqs sequences of max_context are too many pages");
        c->map = std::make_unique<PageMap>((int)num_pages, (int)page_size, (int)max_seqs, (int)c->max_pages);
        OnDevice on(device);
        const size_t meta = 2 * max_seqs + 1 + max_seqs * c->max_pages;
        // a compaction's two tables, its rows' offsets and the rows of a sequence at its longest at least
        c->list_ints = 2 * max_seqs * c->max_pages + max_seqs + 1 + c->max_pages * page_size;
        c->staging.init(meta > c->list_ints ? meta : c->list_ints);
        c->ws_bytes = cactus_cuda_kv4_attention_workspace(max_seqs, max_tokens, num_q_heads, num_kv_heads, head_dim);
        cu(cudaMalloc(&c->pool, num_layers * num_pages * c->page_bytes), "pool");
        cu(cudaMalloc(&c->meta, meta * 4), "batch metadata");
        cu(cudaMalloc(&c->lists, c->list_ints * 4), "page lists");
        cu(cudaMalloc(&c->ws, c->ws_bytes), "workspace");
        cu(cudaMemset(c->ws, 0, c->ws_bytes), "workspace");
        cu(cudaDeviceSynchronize(), "workspace");
        return c.release();
    } catch (const std::exception& e) {
        abi_fail(CB_ERR_ARG, std::string("kv4_create: ") + e.what());
    } catch (...) {
        abi_fail(CB_ERR_ARG, "kv4_create: unknown error");
    }
    cudaGetLastError();  // a failed allocation is this call's alone
    return nullptr;
}

CB_API void cactus_kv4_destroy(cactus_kv4_t cache) { delete static_cast<Cache*>(cache); }

CB_API int cactus_kv4_begin(cactus_kv4_t cache, const int32_t* seqs, const int32_t* new_rows, size_t num_seqs,
                            void* stream) {
    return guarded(cache, "kv4_begin", [&](Cache& c) {
        require(seqs && new_rows && num_seqs >= 1 && num_seqs <= c.max_seqs, "bad list of sequences");
        const std::vector<int> ids = ints(seqs, num_seqs), counts = ints(new_rows, num_seqs);
        size_t total = 0, longest = 0;
        for (int n : counts) {
            require(n >= 0, "a negative number of rows");
            total += (size_t)n;
            longest = longest > (size_t)n ? longest : (size_t)n;
        }
        require(total <= c.max_tokens, "more rows than max_tokens");
        const cudaStream_t st = stream_of(stream);
        const auto copies = c.map->grow(ids, counts);
        c.batch = 0;  // no batch if anything fails from here
        if (!copies.empty()) {
            std::vector<int> v;
            for (const auto& p : copies) v.push_back(p.first);
            for (const auto& p : copies) v.push_back(p.second);
            c.staging.send(v, c.lists, st);
            const int rc = cactus_cuda_kv_copy_pages(c.pool, c.num_pages, c.page_bytes, c.page_bytes, c.layers,
                                                     c.num_pages * c.page_bytes, c.lists, c.lists + copies.size(),
                                                     copies.size(), stream);
            if (rc) return rc;
        }
        size_t width = 1;
        for (int id : ids) width = std::max(width, c.map->pages(id).size());
        std::vector<int> v(2 * c.max_seqs + 1 + num_seqs * width, -1);
        v[0] = 0;
        for (size_t i = 0; i < num_seqs; ++i) {
            v[i + 1] = v[i] + counts[i];
            v[c.max_seqs + 1 + i] = c.map->length(ids[i]);
            const std::vector<int>& pages = c.map->pages(ids[i]);
            std::copy(pages.begin(), pages.end(), v.begin() + 2 * c.max_seqs + 1 + i * width);
        }
        c.staging.send(v, c.meta, st);
        c.batch = num_seqs;
        c.batch_tokens = total;
        c.batch_longest = longest;
        c.batch_pages = width;
        return (int)CB_OK;
    });
}

CB_API int cactus_kv4_append(cactus_kv4_t cache, size_t layer, const uint16_t* keys, const uint16_t* values,
                             size_t row_stride, void* stream) {
    return guarded(cache, "kv4_append", [&](Cache& c) {
        require(layer < c.layers && c.batch, "no such layer, or no batch begun");
        stream_of(stream);
        return cactus_cuda_kv4_append(keys, values, row_stride, c.offsets(), c.lens(), c.table(), c.batch_pages,
                                      c.layer_pool(layer), c.num_pages, c.page_bytes, c.batch, c.batch_tokens, c.page,
                                      c.hkv, c.d, c.g, stream);
    });
}

CB_API int cactus_kv4_rope_append(cactus_kv4_t cache, size_t layer, const uint16_t* queries, size_t query_stride,
                                  uint16_t* rotated, size_t rotated_stride, const uint16_t* keys,
                                  const uint16_t* values, size_t row_stride, const float* rope_table,
                                  size_t num_positions, size_t rotary_dim, const uint16_t* q_weight,
                                  const uint16_t* k_weight, float eps, void* stream) {
    return guarded(cache, "kv4_rope_append", [&](Cache& c) {
        require(layer < c.layers && c.batch, "no such layer, or no batch begun");
        stream_of(stream);
        return cactus_cuda_kv4_rope_append(queries, query_stride, rotated, rotated_stride, keys, values, row_stride,
                                           rope_table, num_positions, rotary_dim, q_weight, k_weight, eps, c.offsets(),
                                           c.lens(), c.table(), c.batch_pages, c.layer_pool(layer), c.num_pages,
                                           c.page_bytes, c.batch, c.batch_tokens, c.hq, c.page, c.hkv, c.d, c.g, stream);
    });
}

CB_API int cactus_kv4_attention(cactus_kv4_t cache, size_t layer, const uint16_t* queries, size_t query_stride,
                                uint16_t* output, float* lse, float scale, size_t window_size, int is_causal,
                                void* stream) {
    return guarded(cache, "kv4_attention", [&](Cache& c) {
        require(layer < c.layers && c.batch, "no such layer, or no batch begun");
        stream_of(stream);
        return cactus_cuda_kv4_attention(queries, query_stride, c.offsets(), c.lens(), c.table(), c.batch_pages,
                                         c.layer_pool(layer), c.num_pages, c.page_bytes, output, lse, c.batch,
                                         c.batch_tokens, c.batch_longest, c.hq, c.page, c.hkv, c.d, c.g, scale,
                                         window_size, is_causal, c.ws, c.ws_bytes, stream);
    });
}

CB_API int cactus_kv4_read(cactus_kv4_t cache, size_t layer, int32_t seq, size_t first, size_t count, uint16_t* keys,
                           uint16_t* values, void* stream) {
    return guarded(cache, "kv4_read", [&](Cache& c) {
        require(layer < c.layers, "no such layer");
        require(first + count >= first && first + count <= (size_t)c.map->length(seq), "rows that the sequence does not have");
        if (count == 0) return (int)CB_OK;
        const cudaStream_t st = stream_of(stream);
        std::vector<int> v = {0, (int)count, (int)first};
        const std::vector<int>& pages = c.map->pages(seq);
        v.insert(v.end(), pages.begin(), pages.end());
        c.staging.send(v, c.lists, st);
        return cactus_cuda_kv4_read(c.layer_pool(layer), c.num_pages, c.page_bytes, c.lists + 3, pages.size(), c.lists,
                                    c.lists + 2, keys, values, 1, count, c.page, c.hkv, c.d, c.g, stream);
    });
}

CB_API int cactus_kv4_fork(cactus_kv4_t cache, const int32_t* src, const int32_t* dst, size_t n) {
    return guarded(cache, "kv4_fork", [&](Cache& c) {
        require((src && dst) || n == 0, "bad list of sequences");
        c.map->fork(ints(src, n), ints(dst, n));
        c.batch = 0;
        return (int)CB_OK;
    });
}

CB_API int cactus_kv4_truncate(cactus_kv4_t cache, int32_t seq, size_t length) {
    return guarded(cache, "kv4_truncate", [&](Cache& c) {
        require(length <= 0x7fffffff, "a length that the sequence does not have");
        c.map->truncate(seq, (int)length);
        c.batch = 0;
        return (int)CB_OK;
    });
}

CB_API int cactus_kv4_free(cactus_kv4_t cache, const int32_t* seqs, size_t n) {
    return guarded(cache, "kv4_free", [&](Cache& c) {
        require(seqs || n == 0, "bad list of sequences");
        for (size_t i = 0; i < n; ++i) c.map->length(seqs[i]);  // all known before any is freed
        for (size_t i = 0; i < n; ++i) c.map->truncate(seqs[i], 0);
        c.batch = 0;
        return (int)CB_OK;
    });
}

CB_API int cactus_kv4_compact(cactus_kv4_t cache, const int32_t* seqs, const int32_t* kept_rows,
                              const int32_t* kept_offsets, size_t num_seqs, void* stream) {
    return guarded(cache, "kv4_compact", [&](Cache& c) {
        require(seqs && kept_offsets && num_seqs >= 1 && num_seqs <= c.max_seqs, "bad list of sequences");
        const std::vector<int> ids = ints(seqs, num_seqs), offs = ints(kept_offsets, num_seqs + 1);
        std::vector<int> counts(num_seqs);
        require(offs[0] == 0, "kept_offsets must start at 0");
        for (size_t i = 0; i < num_seqs; ++i) {
            counts[i] = offs[i + 1] - offs[i];
            require(counts[i] >= 0, "kept_offsets must rise");
        }
        const size_t kept = (size_t)offs.back();
        require(kept_rows || kept == 0, "null kept_rows");
        for (size_t i = 0; i < num_seqs; ++i) {
            const int len = c.map->length(ids[i]);
            for (int j = offs[i]; j < offs[i + 1]; ++j)
                require(kept_rows[j] >= 0 && kept_rows[j] < len, "a kept row that the sequence does not have");
        }
        const cudaStream_t st = stream_of(stream);
        const auto old = c.map->renew(ids, counts);
        c.batch = 0;
        // as many sequences at a time as the lists have room for, at least one (no sequence keeps more rows than
        // its pages can hold); all new pages are taken by now, so none of them is read later
        const size_t w = c.max_pages;
        for (size_t from = 0, to; from < num_seqs; from = to) {
            auto ints_of = [&](size_t end) { return 2 * (end - from) * w + (end - from) + 1 + (size_t)(offs[end] - offs[from]); };
            for (to = from + 1; to < num_seqs && ints_of(to + 1) <= c.list_ints;) ++to;
            const size_t n = to - from, rows = (size_t)(offs[to] - offs[from]);
            if (rows == 0) continue;
            std::vector<int> v(2 * n * w, -1);
            for (size_t i = 0; i < n; ++i) {
                const std::vector<int>& now = c.map->pages(ids[from + i]);
                std::copy(old[from + i].begin(), old[from + i].end(), v.begin() + i * w);
                std::copy(now.begin(), now.end(), v.begin() + (n + i) * w);
            }
            for (size_t i = from; i <= to; ++i) v.push_back(offs[i] - offs[from]);
            v.insert(v.end(), kept_rows + offs[from], kept_rows + offs[to]);
            c.staging.send(v, c.lists, st);
            const int* at = c.lists + 2 * n * w;
            const int rc = cactus_cuda_kv4_compact(c.pool, c.num_pages, c.page_bytes, c.layers, c.num_pages * c.page_bytes,
                                                   c.lists, c.lists + n * w, w, at + n + 1, at, n, rows, c.page, c.hkv, c.d,
                                                   c.g, stream);
            if (rc) return rc;
        }
        return (int)CB_OK;
    });
}

CB_API int cactus_kv4_length(cactus_kv4_t cache, int32_t seq) {
    int len = 0;
    const int rc = guarded(cache, "kv4_length", [&](Cache& c) {
        len = c.map->length(seq);
        return (int)CB_OK;
    });
    return rc ? rc : len;
}

CB_API int cactus_kv4_info(cactus_kv4_t cache, size_t* out4) {
    return guarded(cache, "kv4_info", [&](Cache& c) {
        require(out4 != nullptr, "null argument");
        out4[0] = c.num_pages;
        out4[1] = (size_t)c.map->free_pages();
        out4[2] = c.page_bytes;
        out4[3] = c.layers * c.num_pages * c.page_bytes;
        return (int)CB_OK;
    });
}

}  // extern "C"
