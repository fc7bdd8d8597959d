// Host side of the paged key/value cache (kv.h): allocation, the plan of a
// step and everything that is checked before a kernel sees a page number.
#include "kv.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <new>
#include <string>

#include "scratch.h"

namespace sq {
namespace {

// a * b, or SIZE_MAX where that does not fit
size_t times(size_t a, size_t b) {
    size_t r;
    return __builtin_mul_overflow(a, b, &r) ? SIZE_MAX : r;
}

int on_device(int device, const char* what) {
    int cur = 0;
    SQ_HIP_CHECK(hipGetDevice(&cur));
    if (cur != device)
        return set_error(SQ_ERR_ARG, std::string(what) + ": the cache is on device " + std::to_string(device) +
                                         ", the current device is " + std::to_string(cur));
    return 0;
}

// at least n bytes at *p, whose contents are lost where it has to grow
int grow(void** p, size_t* size, size_t n) {
    if (*size >= n) return 0;
    if (*p) (void)hipFree(*p);
    *p = nullptr;
    *size = 0;
    SQ_HIP_CHECK(device_alloc(p, n));
    *size = n;
    return 0;
}

}  // namespace

int kv_pool_create(size_t n_layers, size_t n_pages, size_t kv_heads, size_t head_dim, const float* inv_freq,
                   size_t half, sq_kv_pool** out) {
    if (n_layers == 0 || n_pages == 0 || kv_heads == 0)
        return set_error(SQ_ERR_SHAPE, "kv_pool: ShapeMismatch (empty pool)");
    if (head_dim != 64 && head_dim != 128)
        return set_error(SQ_ERR_UNSUPPORTED, "kv_pool: head_dim must be 64 or 128");
    if (half > head_dim / 2) return set_error(SQ_ERR_SHAPE, "kv_pool: ShapeMismatch (more frequencies than pairs)");
    if (half && !inv_freq) return set_error(SQ_ERR_ARG, "kv_pool: null inv_freq");
    for (size_t j = 0; j < half; j++)
        if (!std::isfinite(inv_freq[j])) return set_error(SQ_ERR_ARG, "kv_pool: an inverse frequency is not finite");
    if (kv_heads > 4096 || n_pages > (size_t)INT32_MAX || n_layers > (size_t)INT32_MAX)
        return set_error(SQ_ERR_SHAPE, "kv_pool: ShapeMismatch (too many heads, pages or layers)");
    const size_t cells = times(times(n_layers, n_pages), kv_heads);
    const size_t bytes = times(cells, 2 * kPage * head_dim), scales = times(cells, sizeof(float2));
    if (bytes == SIZE_MAX || scales == SIZE_MAX)
        return set_error(SQ_ERR_SHAPE, "kv_pool: ShapeMismatch (size overflows)");
    sq_kv_pool* p = new (std::nothrow) sq_kv_pool();
    if (!p) return set_error(SQ_ERR_ARG, "kv_pool: out of host memory");
    p->n_layers = n_layers;
    p->n_pages = n_pages;
    p->kv_heads = kv_heads;
    p->head_dim = head_dim;
    p->half = half;
    auto fill = [&]() -> int {
        SQ_HIP_CHECK(hipGetDevice(&p->device));
        SQ_HIP_CHECK(device_alloc((void**)&p->bytes, bytes));
        SQ_HIP_CHECK(device_alloc((void**)&p->scales, scales));
        // (a page that no call has written holds zeros, whatever its bytes)
        SQ_HIP_CHECK(hipMemset(p->scales, 0, scales));
        if (half) {
            SQ_HIP_CHECK(device_alloc((void**)&p->inv_freq, half * sizeof(float)));
            SQ_HIP_CHECK(hipMemcpy(p->inv_freq, inv_freq, half * sizeof(float), hipMemcpyHostToDevice));
        }
        SQ_HIP_CHECK(hipStreamSynchronize(nullptr));
        return 0;
    };
    if (int st = fill()) {
        kv_pool_destroy(p);
        return st;
    }
    *out = p;
    return 0;
}

void kv_pool_destroy(sq_kv_pool* p) {
    if (!p) return;
    if (p->bytes) (void)hipFree(p->bytes);
    if (p->scales) (void)hipFree(p->scales);
    if (p->inv_freq) (void)hipFree(p->inv_freq);
    delete p;
}

int kv_plan_create(const sq_kv_pool* pool, sq_kv_plan** out) {
    if (int st = on_device(pool->device, "kv_plan")) return st;
    sq_kv_plan* plan = new (std::nothrow) sq_kv_plan();
    if (!plan) return set_error(SQ_ERR_ARG, "kv_plan: out of host memory");
    plan->pool = pool;
    hipError_t e = hipHostMalloc((void**)&plan->bad, 64, hipHostMallocDefault);
    if (e != hipSuccess) {
        (void)hipGetLastError();
        plan->bad = nullptr;
        kv_plan_destroy(plan);
        return set_error(SQ_ERR_HIP, std::string("hipHostMalloc: ") + hipGetErrorString(e));
    }
    *plan->bad = 0;
    *out = plan;
    return 0;
}

void kv_plan_destroy(sq_kv_plan* plan) {
    if (!plan) return;
    if (plan->dev) (void)hipFree(plan->dev);
    if (plan->rope) (void)hipFree(plan->rope);
    if (plan->bad) (void)hipHostFree(plan->bad);
    delete plan;
}

static int fill_plan(sq_kv_plan* plan, size_t n_seqs, const uint32_t* past, const uint32_t* n_new,
                     const uint32_t* tables, size_t table_stride) {
    const sq_kv_pool& pool = *plan->pool;
    size_t rows = 0, n_pages = 0, n_items = 0;
    for (size_t i = 0; i < n_seqs; i++) {
        const size_t len = (size_t)past[i] + n_new[i];
        const size_t pages = (len + kPage - 1) / kPage;
        if (len > (size_t)INT32_MAX - kPage)
            return set_error(SQ_ERR_SHAPE, "kv_plan: ShapeMismatch (sequence too long)");
        if (pages > table_stride) return set_error(SQ_ERR_SHAPE, "kv_plan: ShapeMismatch (a page table is too short)");
        rows += n_new[i];
        n_pages += pages;
        if (n_new[i]) n_items += pages - past[i] / kPage;
    }
    if (rows > (size_t)INT32_MAX / 4096 || n_pages > (size_t)INT32_MAX)
        return set_error(SQ_ERR_SHAPE, "kv_plan: ShapeMismatch (too many rows or pages)");
    std::vector<KvSeq> seqs(n_seqs);
    const size_t off_items = n_seqs * sizeof(KvSeq), off_pages = off_items + n_items * sizeof(KvItem);
    std::vector<uint8_t> host(off_pages + n_pages * sizeof(int) + 16);
    KvItem* items = (KvItem*)(host.data() + off_items);
    int* pages = (int*)(host.data() + off_pages);
    size_t row = 0, page = 0, item = 0;
    for (size_t i = 0; i < n_seqs; i++) {
        seqs[i] = KvSeq{(int)past[i], (int)n_new[i], (int)row, (int)page};
        const uint32_t* table = tables + i * table_stride;
        const int len = (int)(past[i] + n_new[i]), n = (len + kPage - 1) / kPage;
        for (int j = 0; j < n; j++) {
            if (table[j] >= pool.n_pages)
                return set_error(SQ_ERR_ARG, "kv_plan: page " + std::to_string(table[j]) + " of sequence " +
                                                 std::to_string(i) + " is past the pool's " +
                                                 std::to_string(pool.n_pages));
            pages[page + j] = (int)table[j];
            const int lo = std::max(j * kPage, (int)past[i]), hi = std::min((j + 1) * kPage, len);
            if (lo < hi)
                items[item++] = KvItem{(int)table[j], (int)row + lo - (int)past[i], lo - j * kPage, hi - lo};
        }
        row += n_new[i];
        page += n;
    }
    // A page that the step writes belongs to one place of one sequence: two
    // writers would race, and a reader would see another sequence's rows.
    // (Pages that are only read may be shared: a common prefix.)
    std::vector<int> written(n_items), all(pages, pages + n_pages);
    for (size_t i = 0; i < n_items; i++) written[i] = items[i].page;
    std::sort(written.begin(), written.end());
    std::sort(all.begin(), all.end());
    for (int w : written) {
        const auto r = std::equal_range(all.begin(), all.end(), w);
        if (r.second - r.first != 1)
            return set_error(SQ_ERR_ARG,
                             "kv_plan: page " + std::to_string(w) + " is written by the step and used twice");
    }
    if (n_seqs) memcpy(host.data(), seqs.data(), n_seqs * sizeof(KvSeq));
    // from here on the plan has no valid step until all of it is in place
    plan->seqs.clear();
    plan->rows = plan->n_items = 0;
    plan->rope_ready = false;
    if (int st = grow((void**)&plan->dev, &plan->dev_size, host.size())) return st;
    SQ_HIP_CHECK(hipMemcpy(plan->dev, host.data(), host.size(), hipMemcpyHostToDevice));
    SQ_HIP_CHECK(hipStreamSynchronize(nullptr));
    plan->off_items = off_items;
    plan->off_pages = off_pages;
    plan->rows = rows;
    plan->n_items = n_items;
    plan->seqs.swap(seqs);
    return 0;
}

int kv_plan_fill(sq_kv_plan* plan, size_t n_seqs, const uint32_t* past, const uint32_t* n_new, const uint32_t* tables,
                 size_t table_stride) {
    if (int st = on_device(plan->pool->device, "kv_plan")) return st;
    if (n_seqs > 65535) return set_error(SQ_ERR_SHAPE, "kv_plan: ShapeMismatch (more than 65535 sequences)");
    if (n_seqs && (!past || !n_new || (!tables && table_stride)))
        return set_error(SQ_ERR_ARG, "kv_plan: null argument");
    try {
        return fill_plan(plan, n_seqs, past, n_new, tables, table_stride);
    } catch (const std::bad_alloc&) {
        return set_error(SQ_ERR_ARG, "kv_plan: out of host memory");
    }
}

int kv_views(sq_kv_plan* plan, size_t layer, bool rotate, const char* what, KvView* kv, KvPlanView* pv) {
    const sq_kv_pool& pool = *plan->pool;
    if (int st = on_device(pool.device, what)) return st;
    if (layer >= pool.n_layers) return set_error(SQ_ERR_SHAPE, std::string(what) + ": ShapeMismatch (no such layer)");
    const size_t cells = layer * pool.n_pages * pool.kv_heads;
    *kv = KvView{pool.bytes + cells * 2 * kPage * pool.head_dim, pool.scales + cells, (int)pool.kv_heads,
                 (int)pool.head_dim};
    *pv = KvPlanView{(const KvSeq*)plan->dev,
                     (const int*)(plan->dev + plan->off_pages),
                     (const KvItem*)(plan->dev + plan->off_items),
                     nullptr,
                     nullptr,
                     (int)plan->seqs.size(),
                     (int)plan->n_items,
                     (int)plan->rows,
                     (int)pool.half};
    if (!rotate || !pool.half || !plan->rows) return 0;
    if (!plan->rope_ready) {
        // (growing frees nothing that a queued launch reads: every call waits for its own)
        const size_t n = plan->rows * pool.half;
        if (int st = grow((void**)&plan->rope, &plan->rope_size, n * (sizeof(double2) + sizeof(float2)))) return st;
        if (int st = launch_kv_rope(nullptr, *pv, pool.inv_freq, (int)plan->rows, plan->rope,
                                    (float2*)(plan->rope + n)))
            return st;
        plan->rope_ready = true;
    }
    pv->rope = plan->rope;
    pv->rope32 = (const float2*)(plan->rope + plan->rows * pool.half);
    return 0;
}

}  // namespace sq
