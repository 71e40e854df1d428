// Host runtime of packed prompts (include/vxk.h, vxk_prompt_*): the plan of a
// batch of sequences and the launches over it.
#include "vxk.h"
#include "vxk_internal.h"

#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <chrono>
#include <cmath>
#include <cstring>
#include <new>
#include <queue>
#include <string>
#include <thread>
#include <vector>

namespace {

thread_local std::string g_prompt_create_error;

struct PromptError {
    vxk_status status;
    std::string message;
};

[[noreturn]] void pfail(vxk_status s, const std::string & m) { throw PromptError{s, m}; }

#define VXK_PCUDA(expr)                                                                 \
    do {                                                                                \
        const cudaError_t e_ = (expr);                                                  \
        if (e_ != cudaSuccess) {                                                        \
            pfail(e_ == cudaErrorMemoryAllocation ? VXK_STATUS_OUT_OF_MEMORY            \
                                                  : VXK_STATUS_BACKEND_ERROR,           \
                  std::string(#expr) + ": " + cudaGetErrorString(e_));                  \
        }                                                                               \
    } while (0)

class PromptDevice {
public:
    explicit PromptDevice(int d) {
        cudaGetDevice(&prev_);
        dev_ = d;
        if (prev_ != d) cudaSetDevice(d);
    }
    ~PromptDevice() {
        if (prev_ != dev_) cudaSetDevice(prev_);
    }

private:
    int prev_ = 0, dev_ = 0;
};

size_t align16(size_t n) { return (n + 15) / 16 * 16; }

constexpr size_t kPlanHead = 16;
constexpr int32_t kKeyTile = 128;

// Tensor map {head_dim, heads, rows} over packed 16-bit rows, boxes of 64 dims x
// box_heads x box_rows, 128-byte swizzle, zero fill behind the last row.
void encode_heads_map(CUtensorMap * map, const void * base, const vxk_prompt_config & c, int32_t heads, int64_t rows,
                      int32_t box_heads, int32_t box_rows) {
    // looked up once, by whichever thread comes first
    static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void * fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess || !fn)
            pfail(VXK_STATUS_BACKEND_ERROR, "cuTensorMapEncodeTiled is not available");
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }();
    const cuuint64_t dims[3] = {(cuuint64_t) c.head_dim, (cuuint64_t) heads, (cuuint64_t) rows};
    const cuuint64_t strides[2] = {(cuuint64_t) c.head_dim * 2, (cuuint64_t) c.head_dim * 2 * (cuuint64_t) heads};
    const cuuint32_t box[3] = {64, (cuuint32_t) box_heads, (cuuint32_t) box_rows};
    const cuuint32_t elem[3] = {1, 1, 1};
    const CUresult r = encode(map, c.dtype == VXK_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                              3, const_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) pfail(VXK_STATUS_BACKEND_ERROR, "cuTensorMapEncodeTiled failed for a packed prompt");
}

}  // namespace

struct vxk_prompt {
    vxk_prompt_config cfg{};
    float2 * table = nullptr;
    uint8_t * d_plan = nullptr;
    uint8_t * h_plan[2] = {nullptr, nullptr};
    cudaEvent_t plan_ev[2] = {nullptr, nullptr};
    int plan_next = 0;
    size_t plan_bytes = 0;
    size_t off_items = 0;       // offsets into the plan; CTA offsets follow its head
    int32_t pack_shift = 0;     // log2 of the query heads in one tile
    int32_t tokens = 0;         // tokens in one tile
    int32_t * d_error = nullptr;
    cudaEvent_t ev_sync = nullptr;
    int sm_count = 0;
    int32_t rows = -1;          // rows of the current plan, -1 before the first
    int64_t last_position = -1; // the largest of its positions
    std::string last_error;
};

namespace {

template <typename F>
vxk_status pguarded(vxk_prompt * p, F && body) {
    try {
        body();
        return VXK_STATUS_OK;
    } catch (const PromptError & e) {
        if (p) p->last_error = e.message;
        return e.status;
    } catch (const std::bad_alloc &) {
        if (p) p->last_error = "host out of memory";
        return VXK_STATUS_OUT_OF_MEMORY;
    } catch (...) {
        if (p) p->last_error = "internal error";
        return VXK_STATUS_INTERNAL_ERROR;
    }
}

void free_prompt(vxk_prompt * p) {
    if (!p) return;
    PromptDevice scope(p->cfg.device);
    if (p->table) cudaFree(p->table);
    if (p->d_plan) cudaFree(p->d_plan);
    for (int i = 0; i < 2; ++i) {
        if (p->h_plan[i]) cudaFreeHost(p->h_plan[i]);
        if (p->plan_ev[i]) cudaEventDestroy(p->plan_ev[i]);
    }
    if (p->d_error) cudaFree(p->d_error);
    if (p->ev_sync) cudaEventDestroy(p->ev_sync);
    delete p;
}

void check_config(const vxk_prompt_config & c) {
    if (c.struct_size < sizeof(vxk_prompt_config)) pfail(VXK_STATUS_INVALID_ARGUMENT, "config struct_size too small");
    if (c.head_dim != 64 && c.head_dim != 128) pfail(VXK_STATUS_INVALID_ARGUMENT, "head_dim must be 64 or 128");
    if (c.n_kv_heads < 1 || c.n_q_heads < 1 || c.n_q_heads % c.n_kv_heads != 0 || c.n_q_heads > 1024)
        pfail(VXK_STATUS_INVALID_ARGUMENT, "n_q_heads must be a multiple of n_kv_heads, at most 1024");
    if (c.max_seqs < 1 || c.max_seqs > (1 << 20)) pfail(VXK_STATUS_INVALID_ARGUMENT, "max_seqs must be in [1, 2^20]");
    if (c.max_rows < 1 || c.max_rows > (1 << 22)) pfail(VXK_STATUS_INVALID_ARGUMENT, "max_rows must be in [1, 2^22]");
    if (c.max_position < 0) pfail(VXK_STATUS_INVALID_ARGUMENT, "max_position must not be negative");
    if (c.dtype != VXK_DTYPE_F16 && c.dtype != VXK_DTYPE_BF16)
        pfail(VXK_STATUS_INVALID_ARGUMENT, "the prompt's type must be F16 or BF16");
    if (!(c.rope_theta > 0.0f) || !std::isfinite(c.rope_theta))
        pfail(VXK_STATUS_INVALID_ARGUMENT, "rope_theta must be positive");
    if (!(c.scale >= 0.0f) || !std::isfinite(c.scale))
        pfail(VXK_STATUS_INVALID_ARGUMENT, "scale must be positive, or 0 for 1/sqrt(head_dim)");
    if (c.causal != 0 && c.causal != 1) pfail(VXK_STATUS_INVALID_ARGUMENT, "causal must be 0 or 1");
    if (c.window < 0 || (c.window > 0 && !c.causal))
        pfail(VXK_STATUS_INVALID_ARGUMENT, "window must not be negative and needs causal");
}

void check_capture(cudaStream_t cs, const char * what) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    VXK_PCUDA(cudaStreamIsCapturing(cs, &st));
    if (st != cudaStreamCaptureStatusNone) pfail(VXK_STATUS_INVALID_STATE, std::string(what) + " inside a stream capture");
}

void check_buffers(const vxk_prompt * p, std::initializer_list<const void *> ptrs) {
    if (p->rows < 0) pfail(VXK_STATUS_INVALID_STATE, "no plan");
    for (const void * a : ptrs) {
        if (!a) pfail(VXK_STATUS_INVALID_ARGUMENT, "null buffer");
        if (reinterpret_cast<uintptr_t>(a) % 16 != 0)
            pfail(VXK_STATUS_INVALID_ARGUMENT, "buffers must be 16-byte aligned");
    }
}

void rope(vxk_prompt * prompt, const float2 * table, const float * q, const float * k, const float * v, void * q16,
          void * k16, void * v16, cudaStream_t cs) {
    const vxk_prompt_config & c = prompt->cfg;
    check_buffers(prompt, {q, k, v, q16, k16, v16});
    if (prompt->rows == 0) return;
    PromptDevice scope(c.device);
    vxk::PromptRopeParams a{};
    a.plan = prompt->d_plan;
    a.table = table;
    a.rows = prompt->rows;
    a.n_q = c.n_q_heads;
    a.n_kv = c.n_kv_heads;
    a.head_dim = c.head_dim;
    a.dtype = (int32_t) c.dtype;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q16 = static_cast<uint16_t *>(q16);
    a.k16 = static_cast<uint16_t *>(k16);
    a.v16 = static_cast<uint16_t *>(v16);
    a.error = prompt->d_error;
    VXK_PCUDA(vxk::launch_prompt_rope(a, cs));
}

}  // namespace

namespace vxk {

int32_t prompt_rope_with(vxk_prompt * prompt, const float2 * table, int32_t table_rows, const float * q, const float * k,
                         const float * v, void * q16, void * k16, void * v16, cudaStream_t stream) {
    return pguarded(prompt, [&] {
        if (prompt->last_position >= table_rows) pfail(VXK_STATUS_INVALID_ARGUMENT, "a position lies behind the table");
        rope(prompt, table, q, k, v, q16, k16, v16, stream);
    });
}

}  // namespace vxk

extern "C" {

vxk_prompt_config vxk_prompt_default_config(void) {
    vxk_prompt_config c{};
    c.struct_size = sizeof(vxk_prompt_config);
    c.api_version = VXK_API_VERSION;
    c.n_q_heads = 32;
    c.n_kv_heads = 8;
    c.head_dim = 128;
    c.max_seqs = 1;
    c.max_rows = 512;
    c.max_position = 8192;
    c.dtype = VXK_DTYPE_F16;
    c.rope_theta = 1000000.0f;
    c.causal = 1;
    return c;
}

vxk_status vxk_prompt_create(const vxk_prompt_config * config, vxk_prompt ** out) {
    if (out) *out = nullptr;
    if (!config || !out) {
        g_prompt_create_error = "null argument";
        return VXK_STATUS_INVALID_ARGUMENT;
    }
    vxk_prompt * p = new (std::nothrow) vxk_prompt();
    if (!p) return VXK_STATUS_OUT_OF_MEMORY;
    const vxk_status st = pguarded(p, [&] {
        const vxk_prompt_config & c = *config;
        check_config(c);
        p->cfg = c;
        int n_dev = 0;
        VXK_PCUDA(cudaGetDeviceCount(&n_dev));
        if (c.device < 0 || c.device >= n_dev) {
            p->cfg.device = 0;
            pfail(VXK_STATUS_INVALID_ARGUMENT, "no such CUDA device");
        }
        PromptDevice scope(c.device);
        VXK_PCUDA(cudaDeviceGetAttribute(&p->sm_count, cudaDevAttrMultiProcessorCount, c.device));
        const int32_t group = c.n_q_heads / c.n_kv_heads;
        while (p->pack_shift < 7 && group % (2 << p->pack_shift) == 0) ++p->pack_shift;
        p->tokens = 128 >> p->pack_shift;
        // a sequence's last item may be a part of one
        const size_t max_items = ((size_t) c.max_rows / (2 * p->tokens) + (size_t) std::min(c.max_seqs, c.max_rows)) *
                                 (size_t) (c.n_q_heads >> p->pack_shift);
        p->off_items = kPlanHead + align16((size_t) (p->sm_count + 1) * sizeof(int32_t));
        p->plan_bytes = p->off_items + max_items * sizeof(int4) + (size_t) c.max_rows * sizeof(int32_t);
        VXK_PCUDA(cudaMalloc(&p->d_plan, p->plan_bytes));
        for (int i = 0; i < 2; ++i) {
            VXK_PCUDA(cudaHostAlloc(reinterpret_cast<void **>(&p->h_plan[i]), p->plan_bytes, cudaHostAllocDefault));
            VXK_PCUDA(cudaEventCreateWithFlags(&p->plan_ev[i], cudaEventDisableTiming));
        }
        VXK_PCUDA(cudaMalloc(&p->d_error, sizeof(int32_t)));
        VXK_PCUDA(cudaMemset(p->d_error, 0, sizeof(int32_t)));
        VXK_PCUDA(cudaEventCreateWithFlags(&p->ev_sync, cudaEventDisableTiming));
        if (c.max_position > 0) {
            VXK_PCUDA(cudaMalloc(&p->table, (size_t) c.max_position * (c.head_dim / 2) * sizeof(float2)));
            VXK_PCUDA(vxk::launch_rope_table(p->table, c.max_position, c.head_dim, std::log((double) c.rope_theta),
                                             nullptr));
            VXK_PCUDA(cudaStreamSynchronize(nullptr));
        }
    });
    if (st != VXK_STATUS_OK) {
        g_prompt_create_error = p->last_error;
        free_prompt(p);
        return st;
    }
    *out = p;
    return VXK_STATUS_OK;
}

void vxk_prompt_destroy(vxk_prompt * prompt) { free_prompt(prompt); }

vxk_status vxk_prompt_last_error(const vxk_prompt * prompt, char * buf, size_t capacity) {
    if (!buf || capacity == 0) return VXK_STATUS_INVALID_ARGUMENT;
    const std::string & m = prompt ? prompt->last_error : g_prompt_create_error;
    const size_t n = std::min(capacity - 1, m.size());
    std::memcpy(buf, m.data(), n);
    buf[n] = '\0';
    return m.size() < capacity ? VXK_STATUS_OK : VXK_STATUS_BUFFER_TOO_SMALL;
}

vxk_status vxk_prompt_plan(vxk_prompt * prompt, const int32_t * n_rows, const int32_t * first_position,
                           int32_t n_seqs, void * cuda_stream) {
    if (!prompt) return VXK_STATUS_INVALID_ARGUMENT;
    return pguarded(prompt, [&] {
        const vxk_prompt_config & c = prompt->cfg;
        if (!n_rows || n_seqs < 1 || n_seqs > c.max_seqs)
            pfail(VXK_STATUS_INVALID_ARGUMENT, "n_seqs must be in [1, max_seqs]");
        int64_t total = 0, furthest = -1;
        for (int32_t i = 0; i < n_seqs; ++i) {
            const int64_t first = first_position ? first_position[i] : 0;
            if (n_rows[i] < 0 || first < 0) pfail(VXK_STATUS_INVALID_ARGUMENT, "negative rows or position");
            if (c.max_position > 0 && n_rows[i] > 0 && first + n_rows[i] > c.max_position)
                pfail(VXK_STATUS_INVALID_ARGUMENT, "a position reaches max_position");
            if (n_rows[i] > 0) furthest = std::max(furthest, first + n_rows[i] - 1);
            total += n_rows[i];
        }
        if (furthest > INT32_MAX) pfail(VXK_STATUS_INVALID_ARGUMENT, "a position does not fit 32 bits");
        if (total > c.max_rows) pfail(VXK_STATUS_INVALID_ARGUMENT, "the plan has more than max_rows rows");
        PromptDevice scope(c.device);
        cudaStream_t cs = static_cast<cudaStream_t>(cuda_stream);
        check_capture(cs, "vxk_prompt_plan");
        const int slot = prompt->plan_next;
        VXK_PCUDA(cudaEventSynchronize(prompt->plan_ev[slot]));
        uint8_t * h = prompt->h_plan[slot];

        // Items with their cost (key tiles, and about two for filling and emptying the
        // pipeline), longest first, each to the CTA with the least work so far.
        struct Work {
            int32_t cost;
            int4 item;
        };
        std::vector<Work> work;
        const int32_t per_item = 2 * prompt->tokens, pack = 1 << prompt->pack_shift;
        int32_t row0 = 0;
        for (int32_t i = 0; i < n_seqs; row0 += n_rows[i], ++i) {
            for (int32_t t0 = 0; t0 < n_rows[i]; t0 += per_item) {
                const int32_t last = c.causal ? std::min(t0 + per_item, n_rows[i]) - 1 : n_rows[i] - 1;
                const int32_t lo = c.window > 0 ? std::max(0, t0 - c.window + 1) / kKeyTile : 0;
                for (int32_t hq = 0; hq < c.n_q_heads; hq += pack)
                    work.push_back({last / kKeyTile + 1 - lo + 2, make_int4(row0, n_rows[i], t0, hq)});
            }
        }
        std::stable_sort(work.begin(), work.end(), [](const Work & a, const Work & b) { return a.cost > b.cost; });
        std::vector<std::vector<int32_t>> mine((size_t) prompt->sm_count);
        using Load = std::pair<int64_t, int32_t>;
        std::priority_queue<Load, std::vector<Load>, std::greater<Load>> load;
        for (int32_t i = 0; i < prompt->sm_count; ++i) load.push({0, i});
        for (size_t w = 0; w < work.size(); ++w) {
            const Load l = load.top();
            load.pop();
            mine[(size_t) l.second].push_back((int32_t) w);
            load.push({l.first + work[w].cost, l.second});
        }
        int32_t * offsets = reinterpret_cast<int32_t *>(h + kPlanHead);
        int4 * items = reinterpret_cast<int4 *>(h + prompt->off_items);
        int32_t at = 0;
        for (int32_t i = 0; i < prompt->sm_count; ++i) {
            offsets[i] = at;
            for (const int32_t w : mine[(size_t) i]) items[at++] = work[(size_t) w].item;
        }
        offsets[prompt->sm_count] = at;
        const size_t off_positions = prompt->off_items + (size_t) at * sizeof(int4);
        int32_t * pos = reinterpret_cast<int32_t *>(h + off_positions);
        for (int32_t i = 0; i < n_seqs; ++i)
            for (int32_t j = 0; j < n_rows[i]; ++j) *pos++ = (first_position ? first_position[i] : 0) + j;
        if (off_positions > (size_t) INT32_MAX) pfail(VXK_STATUS_INVALID_ARGUMENT, "the plan is too large");
        const int32_t head[4] = {at, (int32_t) total, n_seqs, (int32_t) off_positions};
        std::memcpy(h, head, sizeof(head));
        VXK_PCUDA(cudaMemcpyAsync(prompt->d_plan, h, off_positions + (size_t) total * sizeof(int32_t),
                                  cudaMemcpyHostToDevice, cs));
        VXK_PCUDA(cudaEventRecord(prompt->plan_ev[slot], cs));
        prompt->plan_next ^= 1;
        prompt->rows = (int32_t) total;
        prompt->last_position = furthest;
    });
}

vxk_status vxk_prompt_rows(const vxk_prompt * prompt, int32_t * out_rows) {
    if (!prompt || !out_rows) return VXK_STATUS_INVALID_ARGUMENT;
    if (prompt->rows < 0) return VXK_STATUS_INVALID_STATE;
    *out_rows = prompt->rows;
    return VXK_STATUS_OK;
}

vxk_status vxk_prompt_rope(vxk_prompt * prompt, const float * q, const float * k, const float * v, void * q16,
                           void * k16, void * v16, void * cuda_stream) {
    if (!prompt) return VXK_STATUS_INVALID_ARGUMENT;
    return pguarded(prompt, [&] {
        if (prompt->cfg.max_position == 0) pfail(VXK_STATUS_INVALID_STATE, "the prompt was created without positions");
        rope(prompt, prompt->table, q, k, v, q16, k16, v16, static_cast<cudaStream_t>(cuda_stream));
    });
}

vxk_status vxk_prompt_attention(vxk_prompt * prompt, const void * q, const void * k, const void * v, void * out,
                                void * cuda_stream) {
    if (!prompt) return VXK_STATUS_INVALID_ARGUMENT;
    return pguarded(prompt, [&] {
        const vxk_prompt_config & c = prompt->cfg;
        check_buffers(prompt, {q, k, v, out});
        if (prompt->rows == 0) return;
        PromptDevice scope(c.device);
        vxk::PromptAttnParams a{};
        a.plan = prompt->d_plan;
        a.off_offsets = (int32_t) kPlanHead;
        a.off_items = (int32_t) prompt->off_items;
        a.rows = prompt->rows;
        a.n_q = c.n_q_heads;
        a.n_kv = c.n_kv_heads;
        a.group = c.n_q_heads / c.n_kv_heads;
        a.pack_shift = prompt->pack_shift;
        a.tokens = prompt->tokens;
        a.out_32 = reinterpret_cast<uintptr_t>(out) % 32 == 0;
        a.head_dim = c.head_dim;
        a.dtype = (int32_t) c.dtype;
        a.causal = c.causal;
        a.window = c.window;
        const double scale = c.scale > 0.0f ? (double) c.scale : 1.0 / std::sqrt((double) c.head_dim);
        a.scale_log2 = (float) (scale * 1.4426950408889634);
        a.v = v;
        a.out = out;
        a.error = prompt->d_error;
        CUtensorMap mq{}, mk{}, mv{};
        encode_heads_map(&mq, q, c, c.n_q_heads, prompt->rows, 1 << prompt->pack_shift, prompt->tokens);
        encode_heads_map(&mk, k, c, c.n_kv_heads, prompt->rows, 1, kKeyTile);
        encode_heads_map(&mv, v, c, c.n_kv_heads, prompt->rows, 1, kKeyTile);
        VXK_PCUDA(vxk::launch_prompt_attention(a, mq, mk, mv, prompt->sm_count, static_cast<cudaStream_t>(cuda_stream)));
    });
}

vxk_status vxk_prompt_sync(vxk_prompt * prompt, void * cuda_stream, int32_t timeout_ms) {
    if (!prompt) return VXK_STATUS_INVALID_ARGUMENT;
    return pguarded(prompt, [&] {
        PromptDevice scope(prompt->cfg.device);
        VXK_PCUDA(cudaEventRecord(prompt->ev_sync, static_cast<cudaStream_t>(cuda_stream)));
        const auto t0 = std::chrono::steady_clock::now();
        while (true) {
            const cudaError_t e = cudaEventQuery(prompt->ev_sync);
            if (e == cudaSuccess) break;
            if (e != cudaErrorNotReady) pfail(VXK_STATUS_BACKEND_ERROR, cudaGetErrorString(e));
            const auto ms =
                std::chrono::duration_cast<std::chrono::milliseconds>(std::chrono::steady_clock::now() - t0).count();
            if (ms > timeout_ms) pfail(VXK_STATUS_TIMEOUT, "stream did not drain within the timeout");
            // poll short waits; sleep between polls after 20 ms
            if (ms < 20)
                std::this_thread::yield();
            else
                std::this_thread::sleep_for(std::chrono::microseconds(50));
        }
        int32_t err = 0;
        VXK_PCUDA(cudaMemcpy(&err, prompt->d_error, sizeof(err), cudaMemcpyDeviceToHost));
        if (err != 0) {
            VXK_PCUDA(cudaMemset(prompt->d_error, 0, sizeof(int32_t)));
            if (err == vxk::kErrPlan)
                pfail(VXK_STATUS_BACKEND_ERROR, "a replayed call met a plan of more rows than it was captured under");
            pfail(VXK_STATUS_BACKEND_ERROR, "prompt kernel reported a device error (bounded wait expired)");
        }
    });
}

}  // extern "C"
