// batch_api.cpp -- the C ABI of include/wick_hip_batch.h: the caches of a batch, the
// plan of its steps and the launches.
//
// A plan lives in one device block: header, tokens, items.  The host writes it into
// pinned memory (two blocks in turn, each behind an event) and copies it on the
// handle's stream, so the kernels queued before still read the plan they were called
// under.  The block, the states and everything else that append and attention use are
// allocated at creation and never move: captured calls stay valid.
#include "wick_hip_batch.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <new>
#include <utility>
#include <vector>

#include "attn_kernels.h"
#include "batch_kernels.h"

struct wick_hip_batch {
    wick_hip_batch_config cfg{};
    wick::BatchLimits lim{};
    int device = 0;
    hipStream_t own_stream = nullptr, stream = nullptr;
    hipEvent_t moved = nullptr;                            // orders two streams (set_stream)
    char *pk = nullptr, *pv = nullptr, *k = nullptr, *v = nullptr;
    char *plan_dev = nullptr;
    size_t plan_bytes = 0, items_at = 0;
    char *plan_host[2] = {};
    hipEvent_t plan_sent[2] = {};
    int plan_slot = 0;
    float *states = nullptr;
    int64_t max_items = 0, state_rows = 0;
    // the current plan
    wick::BatchHeader head{};
    bool planned = false;
    int shape = 0;  // of the last plan
    // the last plans' shapes, the newest at the end: a step of prompts between steps of answers
    // leaves the answers' number, and the graphs captured under it, as they were
    struct Shape {
        std::vector<int> t;
        int number;
    };
    std::vector<Shape> shapes;
    int numbers = 0;  // given so far; none is given twice
    // staging of the host-array calls
    float *stage = nullptr;
    size_t stage_floats = 0;

    size_t esize() const { return cfg.type == WICK_HIP_BATCH_BF16 ? 2 : 4; }
    size_t prefix_layer() const { return (size_t)cfg.kv_heads * cfg.prefix_capacity * cfg.head_dim * esize(); }
    size_t own_layer() const {
        return (size_t)cfg.sequences * cfg.kv_heads * cfg.capacity * cfg.head_dim * esize();
    }
    const wick::BatchHeader *head_dev() const { return reinterpret_cast<const wick::BatchHeader *>(plan_dev); }
    const wick::BatchToken *tokens_dev() const {
        return reinterpret_cast<const wick::BatchToken *>(plan_dev + sizeof(wick::BatchHeader));
    }
    const wick::BatchItem *items_dev() const { return reinterpret_cast<const wick::BatchItem *>(plan_dev + items_at); }
};

namespace {

using wick::set_error;

constexpr size_t kShapes = 32;  // plans whose shapes are known again

int hip_fail(hipError_t e, const char *what) {
    return set_error(e == hipErrorOutOfMemory ? WICK_HIP_ENOMEM : WICK_HIP_EHIP, "%s: %s", what, hipGetErrorString(e));
}

#define HIP_TRY(expr)                                     \
    do {                                                  \
        hipError_t e_ = (expr);                           \
        if (e_ != hipSuccess) return hip_fail(e_, #expr); \
    } while (0)

// The handle's device for the length of a call, whichever is current.
class OnDevice {
  public:
    explicit OnDevice(int device) {
        if (hipGetDevice(&before_) != hipSuccess) before_ = device;
        if (before_ != device) rc = hipSetDevice(device);
        changed_ = before_ != device;
    }
    ~OnDevice() {
        if (changed_) (void)hipSetDevice(before_);
    }
    hipError_t rc = hipSuccess;

  private:
    int before_ = 0;
    bool changed_ = false;
};

#define ON_DEVICE(b)         \
    OnDevice on_((b)->device); \
    if (on_.rc != hipSuccess) return hip_fail(on_.rc, "hipSetDevice")

// For the length of a call: what it waits for or allocates would, in the default mode, end a
// capture in progress on another handle's or program's stream.
class BesideCaptures {
  public:
    BesideCaptures() { changed_ = hipThreadExchangeStreamCaptureMode(&mode_) == hipSuccess; }
    ~BesideCaptures() {
        if (changed_) (void)hipThreadExchangeStreamCaptureMode(&mode_);
    }

  private:
    hipStreamCaptureMode mode_ = hipStreamCaptureModeRelaxed;
    bool changed_;
};

bool capturing(hipStream_t s) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &st) != hipSuccess) {
        (void)hipGetLastError();
        return true;
    }
    return st != hipStreamCaptureStatusNone;
}

int check_layer(const wick_hip_batch *b, int layer) {
    if (!b) return set_error(WICK_HIP_EINVAL, "null batch handle");
    if (layer < 0 || layer >= b->cfg.layers)
        return set_error(WICK_HIP_EINVAL, "layer %d out of range [0, %d)", layer, b->cfg.layers);
    return WICK_HIP_OK;
}

int check_aligned(const void *p, const char *what) {
    if (!p) return set_error(WICK_HIP_EINVAL, "null %s", what);
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return set_error(WICK_HIP_EINVAL, "%s is not 16-byte aligned", what);
    return WICK_HIP_OK;
}

int check_planned(const wick_hip_batch *b) {
    if (!b->planned) return set_error(WICK_HIP_EINVAL, "no plan (call wick_hip_batch_plan first)");
    return WICK_HIP_OK;
}

int check_config(const wick_hip_batch_config &c) {
    if (c.layers < 1 || c.kv_heads < 1 || c.sequences < 1 || c.capacity < 1 || c.max_tokens < 1)
        return set_error(WICK_HIP_EINVAL, "layers, kv_heads, sequences, capacity and max_tokens must be >= 1");
    if (c.heads < 1 || c.heads % c.kv_heads != 0)
        return set_error(WICK_HIP_EINVAL, "heads (%d) must be a positive multiple of kv_heads (%d)", c.heads, c.kv_heads);
    if (c.kv_heads > 65535) return set_error(WICK_HIP_EINVAL, "kv_heads must be at most 65535");
    if (c.head_dim != 16 && c.head_dim != 32 && c.head_dim != 64 && c.head_dim != 128)
        return set_error(WICK_HIP_EINVAL, "head_dim %d not supported (16, 32, 64, 128)", c.head_dim);
    if (c.prefix_capacity < 0) return set_error(WICK_HIP_EINVAL, "prefix_capacity must be >= 0");
    if (c.type != WICK_HIP_BATCH_F32 && c.type != WICK_HIP_BATCH_BF16)
        return set_error(WICK_HIP_EINVAL, "unknown cache type %d", c.type);
    // positions and rows are 32-bit numbers with room for a step more
    if (c.capacity > (1 << 30) || c.prefix_capacity > (1 << 30))
        return set_error(WICK_HIP_EINVAL, "capacities must be at most 2^30");
    if ((long long)c.max_tokens * (c.heads / c.kv_heads) > (1 << 30))
        return set_error(WICK_HIP_EINVAL, "max_tokens * heads / kv_heads must be at most 2^30");
    if ((long long)c.max_tokens > (long long)c.sequences * c.capacity)
        return set_error(WICK_HIP_EINVAL, "max_tokens %d exceeds the %d sequences' %d positions", c.max_tokens, c.sequences,
                         c.capacity);
    return WICK_HIP_OK;
}

int stage_for(wick_hip_batch *b, size_t floats) {
    if (capturing(b->stream)) return set_error(WICK_HIP_EINVAL, "a host-array call on a stream that is being captured");
    if (floats <= b->stage_floats) return WICK_HIP_OK;
    HIP_TRY(hipStreamSynchronize(b->stream));
    if (b->stage) (void)hipFree(b->stage);
    b->stage = nullptr;
    b->stage_floats = 0;
    HIP_TRY(hipMalloc(&b->stage, floats * sizeof(float)));
    b->stage_floats = floats;
    return WICK_HIP_OK;
}

// What one HIP-side allocation needs; false where its size has no room in a size_t.
bool product(size_t *out, std::initializer_list<size_t> f) {
    size_t n = 1;
    for (size_t x : f)
        if (__builtin_mul_overflow(n, x, &n)) return false;
    *out = n;
    return true;
}

int set_up(wick_hip_batch *b) {
    const wick_hip_batch_config &c = b->cfg;
    HIP_TRY(hipGetDevice(&b->device));
    hipDeviceProp_t prop;
    HIP_TRY(hipGetDeviceProperties(&prop, b->device));
    if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0)
        return set_error(WICK_HIP_EDEVICE, "device %d is %s; this library is built for gfx950", b->device, prop.gcnArchName);
    b->lim.group = c.heads / c.kv_heads;
    b->lim.kv_heads = c.kv_heads;
    b->lim.sequences = c.sequences;
    b->lim.capacity = c.capacity;
    b->lim.prefix_capacity = c.prefix_capacity;
    b->lim.max_tokens = c.max_tokens;
    b->lim.cus = prop.multiProcessorCount;
    b->lim.few = wick::batch_few(c.type == WICK_HIP_BATCH_BF16);
    b->max_items = wick::batch_max_items(b->lim);
    b->state_rows = wick::batch_max_state_rows(b->lim);
    // a launch holds 2^32 threads, and state rows are 32-bit numbers
    if (b->max_items * c.kv_heads > (1 << 23) || b->state_rows > INT_MAX / 2)
        return set_error(WICK_HIP_EINVAL, "max_tokens %d is too large", c.max_tokens);
    b->items_at = sizeof(wick::BatchHeader) + (size_t)c.max_tokens * sizeof(wick::BatchToken);
    b->items_at = (b->items_at + 63) / 64 * 64;
    b->plan_bytes = b->items_at + (size_t)b->max_items * sizeof(wick::BatchItem);
    b->shapes.reserve(kShapes);
    HIP_TRY(hipStreamCreateWithFlags(&b->own_stream, hipStreamNonBlocking));
    b->stream = b->own_stream;
    HIP_TRY(hipEventCreateWithFlags(&b->moved, hipEventDisableTiming));
    for (int i = 0; i < 2; i++) {
        HIP_TRY(hipEventCreateWithFlags(&b->plan_sent[i], hipEventDisableTiming));
        HIP_TRY(hipHostMalloc(reinterpret_cast<void **>(&b->plan_host[i]), b->plan_bytes, hipHostMallocDefault));
    }
    HIP_TRY(hipMalloc(&b->plan_dev, b->plan_bytes));
    HIP_TRY(hipMemsetAsync(b->plan_dev, 0, sizeof(wick::BatchHeader), b->stream));
    size_t bytes;
    if (!product(&bytes, {(size_t)c.kv_heads, (size_t)b->state_rows, (size_t)c.head_dim + 2, sizeof(float)}))
        return set_error(WICK_HIP_ENOMEM, "the states' size overflows");
    HIP_TRY(hipMalloc(&b->states, bytes));
    struct {
        char **p;
        bool own;
    } caches[] = {{&b->pk, false}, {&b->pv, false}, {&b->k, true}, {&b->v, true}};
    for (auto &x : caches) {
        const size_t L = (size_t)c.layers, H = (size_t)c.kv_heads, D = (size_t)c.head_dim;
        const bool ok = x.own ? product(&bytes, {L, (size_t)c.sequences, H, (size_t)c.capacity, D, b->esize()})
                              : product(&bytes, {L, H, (size_t)c.prefix_capacity, D, b->esize()});
        if (!ok) return set_error(WICK_HIP_ENOMEM, "the caches' size overflows");
        if (bytes == 0) continue;
        HIP_TRY(hipMalloc(x.p, bytes));
        HIP_TRY(hipMemsetAsync(*x.p, 0, bytes, b->stream));
    }
    HIP_TRY(hipStreamSynchronize(b->stream));
    return WICK_HIP_OK;
}

}  // namespace

extern "C" {

int wick_hip_batch_create(const wick_hip_batch_config *cfg, wick_hip_batch **out) {
    if (!cfg || !out) return set_error(WICK_HIP_EINVAL, "null argument");
    *out = nullptr;
    if (int rc = check_config(*cfg)) return rc;
    BesideCaptures beside;
    int ndev = 0;
    if (hipGetDeviceCount(&ndev) != hipSuccess || ndev < 1) return set_error(WICK_HIP_EDEVICE, "no HIP device");
    wick_hip_batch *b = new (std::nothrow) wick_hip_batch;
    if (!b) return set_error(WICK_HIP_ENOMEM, "out of host memory");
    b->cfg = *cfg;
    int rc;
    try {
        rc = set_up(b);
    } catch (const std::bad_alloc &) {
        rc = set_error(WICK_HIP_ENOMEM, "out of host memory");
    }
    if (rc) {
        wick_hip_batch_destroy(b);
        return rc;
    }
    *out = b;
    return WICK_HIP_OK;
}

void wick_hip_batch_destroy(wick_hip_batch *b) {
    if (!b) return;
    OnDevice on(b->device);
    BesideCaptures beside;
    if (b->stream) (void)hipStreamSynchronize(b->stream);
    for (void *p : {(void *)b->pk, (void *)b->pv, (void *)b->k, (void *)b->v, (void *)b->plan_dev, (void *)b->states,
                    (void *)b->stage})
        if (p) (void)hipFree(p);
    for (int i = 0; i < 2; i++) {
        if (b->plan_host[i]) (void)hipHostFree(b->plan_host[i]);
        if (b->plan_sent[i]) (void)hipEventDestroy(b->plan_sent[i]);
    }
    if (b->moved) (void)hipEventDestroy(b->moved);
    if (b->own_stream) (void)hipStreamDestroy(b->own_stream);
    delete b;
}

int wick_hip_batch_load_prefix(wick_hip_batch *b, const wick_hip_kv *kv, int len) {
    if (!b) return set_error(WICK_HIP_EINVAL, "null batch handle");
    wick::KvInfo info;
    if (!wick::kv_info(kv, &info)) return set_error(WICK_HIP_EINVAL, "null cache handle");
    const wick_hip_batch_config &c = b->cfg;
    if (info.layers != c.layers || info.kv_heads != c.kv_heads || info.head_dim != c.head_dim)
        return set_error(WICK_HIP_EINVAL, "the cache has %d layers of %d x %d, the batch %d of %d x %d", info.layers,
                         info.kv_heads, info.head_dim, c.layers, c.kv_heads, c.head_dim);
    if (len < 0 || len > info.capacity || len > c.prefix_capacity)
        return set_error(WICK_HIP_EINVAL, "%d positions exceed the cache's %d or the prefix's %d", len, info.capacity,
                         c.prefix_capacity);
    if (len == 0) return WICK_HIP_OK;
    const float *k, *v;
    int device;
    wick::kv_layer(kv, 0, &k, &v, &device);
    if (device != b->device) return set_error(WICK_HIP_EINVAL, "the cache is on device %d, the batch on %d", device, b->device);
    ON_DEVICE(b);
    BesideCaptures beside;
    if (capturing(b->stream) || capturing(info.stream))
        return set_error(WICK_HIP_EINVAL, "wick_hip_batch_load_prefix on a stream that is being captured");
    HIP_TRY(hipStreamSynchronize(info.stream));
    for (int l = 0; l < c.layers; l++) {
        wick::kv_layer(kv, l, &k, &v, &device);
        HIP_TRY(wick::launch_batch_load(c.head_dim, c.type, k, info.capacity, b->pk + l * b->prefix_layer(),
                                        c.prefix_capacity, c.kv_heads, len, b->stream));
        HIP_TRY(wick::launch_batch_load(c.head_dim, c.type, v, info.capacity, b->pv + l * b->prefix_layer(),
                                        c.prefix_capacity, c.kv_heads, len, b->stream));
    }
    HIP_TRY(hipStreamSynchronize(b->stream));
    return WICK_HIP_OK;
}

int wick_hip_batch_write_prefix_device(wick_hip_batch *b, int layer, int start, int t, const float *k_dev,
                                       const float *v_dev) {
    if (int rc = check_layer(b, layer)) return rc;
    if (t < 1) return set_error(WICK_HIP_EINVAL, "t must be >= 1 (got %d)", t);
    if (start < 0 || (long long)start + t > b->cfg.prefix_capacity)
        return set_error(WICK_HIP_EINVAL, "positions %d..%lld exceed the prefix capacity %d", start, (long long)start + t,
                         b->cfg.prefix_capacity);
    if (int rc = check_aligned(k_dev, "k_dev")) return rc;
    if (int rc = check_aligned(v_dev, "v_dev")) return rc;
    ON_DEVICE(b);
    wick::BatchAppendArgs a{};
    a.ksrc = k_dev;
    a.vsrc = v_dev;
    a.k = b->pk + layer * b->prefix_layer();
    a.v = b->pv + layer * b->prefix_layer();
    a.capacity = b->cfg.prefix_capacity;
    a.kv_heads = b->cfg.kv_heads;
    a.total = t;
    a.start = start;
    HIP_TRY(wick::launch_batch_append(b->cfg.head_dim, b->cfg.type, a, b->stream));
    return WICK_HIP_OK;
}

int wick_hip_batch_plan(wick_hip_batch *b, const int *start, const int *t, int prefix) {
    if (!b) return set_error(WICK_HIP_EINVAL, "null batch handle");
    if (!start || !t) return set_error(WICK_HIP_EINVAL, "null start or t");
    const wick_hip_batch_config &c = b->cfg;
    if (prefix < 0 || prefix > c.prefix_capacity)
        return set_error(WICK_HIP_EINVAL, "prefix %d exceeds the prefix capacity %d", prefix, c.prefix_capacity);
    long long total = 0;
    for (int s = 0; s < c.sequences; s++) {
        if (t[s] < 0 || start[s] < 0 || (long long)start[s] + t[s] > c.capacity)
            return set_error(WICK_HIP_EINVAL, "sequence %d: positions %d..%lld exceed the capacity %d", s, start[s],
                             (long long)start[s] + t[s], c.capacity);
        total += t[s];
    }
    if (total > c.max_tokens)
        return set_error(WICK_HIP_EINVAL, "%lld tokens exceed max_tokens %d", total, c.max_tokens);
    ON_DEVICE(b);
    BesideCaptures beside;
    if (capturing(b->stream)) return set_error(WICK_HIP_EINVAL, "wick_hip_batch_plan on a stream that is being captured");
    try {
        wick::BatchPlan p = wick::batch_plan(b->lim, start, t, prefix);
        if (p.head.items > b->max_items || p.head.items > p.head.most_items || p.state_rows > b->state_rows)
            return set_error(WICK_HIP_EHIP, "internal: the plan has %d items and %lld state rows", p.head.items,
                             (long long)p.state_rows);
        const int slot = b->plan_slot;
        HIP_TRY(hipEventSynchronize(b->plan_sent[slot]));
        // captured calls depend on the tokens of every sequence, and on nothing else of a plan
        auto known = std::find_if(b->shapes.begin(), b->shapes.end(), [&](const wick_hip_batch::Shape &x) {
            return std::memcmp(x.t.data(), t, c.sequences * sizeof(int)) == 0;
        });
        if (known == b->shapes.end()) {
            wick_hip_batch::Shape x{std::vector<int>(t, t + c.sequences), ++b->numbers};
            if (b->shapes.size() == kShapes) b->shapes.erase(b->shapes.begin());
            b->shapes.push_back(std::move(x));
        } else {
            std::rotate(known, known + 1, b->shapes.end());
        }
        b->shape = p.head.shape = b->shapes.back().number;
        char *h = b->plan_host[slot];
        const size_t tokens = p.tokens.size() * sizeof(wick::BatchToken), items = p.items.size() * sizeof(wick::BatchItem);
        std::memcpy(h, &p.head, sizeof p.head);
        if (tokens) std::memcpy(h + sizeof p.head, p.tokens.data(), tokens);
        if (items) std::memcpy(h + b->items_at, p.items.data(), items);
        b->planned = false;  // until both copies are queued
        HIP_TRY(hipMemcpyAsync(b->plan_dev, h, sizeof p.head + tokens, hipMemcpyHostToDevice, b->stream));
        if (items)
            HIP_TRY(hipMemcpyAsync(b->plan_dev + b->items_at, h + b->items_at, items, hipMemcpyHostToDevice, b->stream));
        HIP_TRY(hipEventRecord(b->plan_sent[slot], b->stream));
        b->plan_slot = 1 - slot;
        b->head = p.head;
        b->planned = true;
    } catch (const std::bad_alloc &) {
        return set_error(WICK_HIP_ENOMEM, "out of host memory");
    }
    return WICK_HIP_OK;
}

int wick_hip_batch_shape(const wick_hip_batch *b) { return b ? b->shape : 0; }

int wick_hip_batch_append_device(wick_hip_batch *b, int layer, const float *k_dev, const float *v_dev) {
    if (int rc = check_layer(b, layer)) return rc;
    if (int rc = check_planned(b)) return rc;
    if (b->head.total == 0) return WICK_HIP_OK;
    if (int rc = check_aligned(k_dev, "k_dev")) return rc;
    if (int rc = check_aligned(v_dev, "v_dev")) return rc;
    ON_DEVICE(b);
    wick::BatchAppendArgs a{};
    a.ksrc = k_dev;
    a.vsrc = v_dev;
    a.k = b->k + layer * b->own_layer();
    a.v = b->v + layer * b->own_layer();
    a.head = b->head_dev();
    a.tokens = b->tokens_dev();
    a.capacity = b->cfg.capacity;
    a.kv_heads = b->cfg.kv_heads;
    a.total = b->head.total;
    a.shape = b->shape;
    HIP_TRY(wick::launch_batch_append(b->cfg.head_dim, b->cfg.type, a, b->stream));
    return WICK_HIP_OK;
}

int wick_hip_batch_attention_device(wick_hip_batch *b, int layer, const float *q_dev, float *att_dev) {
    if (int rc = check_layer(b, layer)) return rc;
    if (int rc = check_planned(b)) return rc;
    if (b->head.total == 0) return WICK_HIP_OK;
    if (int rc = check_aligned(q_dev, "q_dev")) return rc;
    if (int rc = check_aligned(att_dev, "att_dev")) return rc;
    ON_DEVICE(b);
    const wick_hip_batch_config &c = b->cfg;
    wick::BatchArgs a{};
    a.q = q_dev;
    a.att = att_dev;
    a.pk = b->pk + layer * b->prefix_layer();
    a.pv = b->pv + layer * b->prefix_layer();
    a.k = b->k + layer * b->own_layer();
    a.v = b->v + layer * b->own_layer();
    a.head = b->head_dev();
    a.tokens = b->tokens_dev();
    a.items = b->items_dev();
    a.state_rows = b->state_rows;
    a.po = b->states;
    a.pm = a.po + (size_t)c.kv_heads * b->state_rows * c.head_dim;
    a.pl = a.pm + (size_t)c.kv_heads * b->state_rows;
    a.prefix_capacity = c.prefix_capacity;
    a.capacity = c.capacity;
    a.group = b->lim.group;
    a.kv_heads = c.kv_heads;
    a.inv_group = wick::batch_inverse(a.group);
    a.inv_kv_heads = wick::batch_inverse(a.kv_heads);
    a.inv_heads = wick::batch_inverse(c.heads);
    a.shape = b->shape;
    a.total = b->head.total;
    a.max_states = b->head.max_states;  // a captured call chooses by its own plan's
    a.scale = (float)(M_LOG2E / std::sqrt((double)c.head_dim));
    // a captured call serves later plans too: those may have more items, or states to join
    // where this one has none
    const bool later = capturing(b->stream);
    const int items = later ? b->head.most_items : b->head.items;
    a.launched = items;
    HIP_TRY(wick::launch_batch_attend(c.head_dim, c.type, a, items * c.kv_heads, b->stream));
    const int merges = later ? b->head.total : b->head.merges;
    if (merges) HIP_TRY(wick::launch_batch_merge(c.head_dim, a, merges, b->stream));
    return WICK_HIP_OK;
}

int wick_hip_batch_append(wick_hip_batch *b, int layer, const float *k, const float *v) {
    if (int rc = check_layer(b, layer)) return rc;
    if (int rc = check_planned(b)) return rc;
    if (b->head.total == 0) return WICK_HIP_OK;
    if (!k || !v) return set_error(WICK_HIP_EINVAL, "null k or v");
    ON_DEVICE(b);
    BesideCaptures beside;
    const size_t n = (size_t)b->head.total * b->cfg.kv_heads * b->cfg.head_dim;
    if (int rc = stage_for(b, 2 * n)) return rc;
    HIP_TRY(hipMemcpyAsync(b->stage, k, n * sizeof(float), hipMemcpyHostToDevice, b->stream));
    HIP_TRY(hipMemcpyAsync(b->stage + n, v, n * sizeof(float), hipMemcpyHostToDevice, b->stream));
    if (int rc = wick_hip_batch_append_device(b, layer, b->stage, b->stage + n)) return rc;
    HIP_TRY(hipStreamSynchronize(b->stream));
    return WICK_HIP_OK;
}

int wick_hip_batch_attention(wick_hip_batch *b, int layer, const float *q, float *att) {
    if (int rc = check_layer(b, layer)) return rc;
    if (int rc = check_planned(b)) return rc;
    if (b->head.total == 0) return WICK_HIP_OK;
    if (!q || !att) return set_error(WICK_HIP_EINVAL, "null q or att");
    ON_DEVICE(b);
    BesideCaptures beside;
    const size_t n = (size_t)b->head.total * b->cfg.heads * b->cfg.head_dim;
    if (int rc = stage_for(b, 2 * n)) return rc;
    HIP_TRY(hipMemcpyAsync(b->stage, q, n * sizeof(float), hipMemcpyHostToDevice, b->stream));
    if (int rc = wick_hip_batch_attention_device(b, layer, b->stage, b->stage + n)) return rc;
    HIP_TRY(hipMemcpyAsync(att, b->stage + n, n * sizeof(float), hipMemcpyDeviceToHost, b->stream));
    HIP_TRY(hipStreamSynchronize(b->stream));
    return WICK_HIP_OK;
}

int wick_hip_batch_read(wick_hip_batch *b, int layer, int seq, int pos0, int n, float *k, float *v) {
    if (int rc = check_layer(b, layer)) return rc;
    const wick_hip_batch_config &c = b->cfg;
    if (seq < -1 || seq >= c.sequences)
        return set_error(WICK_HIP_EINVAL, "sequence %d out of range [-1, %d)", seq, c.sequences);
    const int capacity = seq < 0 ? c.prefix_capacity : c.capacity;
    if (n < 1 || pos0 < 0 || (long long)pos0 + n > capacity)
        return set_error(WICK_HIP_EINVAL, "positions %d..%lld exceed the capacity %d", pos0, (long long)pos0 + n, capacity);
    ON_DEVICE(b);
    BesideCaptures beside;
    const size_t floats = (size_t)n * c.kv_heads * c.head_dim;
    if (int rc = stage_for(b, floats)) return rc;
    for (int x = 0; x < 2; x++) {
        float *dst = x ? v : k;
        if (!dst) continue;
        const char *src = seq < 0 ? (x ? b->pv : b->pk) + layer * b->prefix_layer()
                                  : (x ? b->v : b->k) + layer * b->own_layer() +
                                        (size_t)seq * (b->own_layer() / c.sequences);
        HIP_TRY(wick::launch_batch_read(c.head_dim, c.type, src, capacity, c.kv_heads, pos0, n, b->stage, b->stream));
        HIP_TRY(hipMemcpyAsync(dst, b->stage, floats * sizeof(float), hipMemcpyDeviceToHost, b->stream));
    }
    HIP_TRY(hipStreamSynchronize(b->stream));
    return WICK_HIP_OK;
}

int wick_hip_batch_set_stream(wick_hip_batch *b, void *stream) {
    if (!b) return set_error(WICK_HIP_EINVAL, "null batch handle");
    hipStream_t to = stream ? static_cast<hipStream_t>(stream) : b->own_stream;
    if (to == b->stream) return WICK_HIP_OK;
    ON_DEVICE(b);
    if (!capturing(b->stream) && !capturing(to)) {
        HIP_TRY(hipEventRecord(b->moved, b->stream));
        HIP_TRY(hipStreamWaitEvent(to, b->moved, 0));
    }
    b->stream = to;
    return WICK_HIP_OK;
}

int wick_hip_batch_synchronize(wick_hip_batch *b) {
    if (!b) return set_error(WICK_HIP_EINVAL, "null batch handle");
    ON_DEVICE(b);
    BesideCaptures beside;
    HIP_TRY(hipStreamSynchronize(b->stream));
    return WICK_HIP_OK;
}

long long wick_hip_batch_scratch_bytes(const wick_hip_batch *b) {
    if (!b) return 0;
    return (long long)(3 * b->plan_bytes + b->stage_floats * sizeof(float) +
                       (size_t)b->cfg.kv_heads * b->state_rows * (b->cfg.head_dim + 2) * sizeof(float));
}

}  // extern "C"
