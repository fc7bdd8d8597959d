// The paged key/value cache in 8 bits: its memory, the plan of one step over
// it, and the layout that the kernels share.
//
// A page holds 64 consecutive positions of one sequence, for every layer and
// KV head, with one f32 scale for its keys and one for its values: the stored
// byte b stands for (b - 128) * scale.  Within a (page, head) the keys come
// first, then the values, each in the order in which a wavefront's 16-byte
// loads hand them to v_mfma_*_16x16x*:
//   keys    in tiles of 16 positions; a tile's load is lane (16 g + i):
//           position i of the tile, dimensions 16 g .. 16 g + 15 (of each 64)
//   values  in tiles of 16 dimensions; lane (16 g + i) has dimension i of the
//           tile and sixteen positions, those with position % 16 in 4 g ..
//           4 g + 3.  That is the set of positions whose scores lane group g
//           holds after the product of the four key tiles with the queries
//           (row 4 g + r of tile t is position 16 t + 4 g + r), in the order
//           4 r + t, so probabilities never cross lanes between the products.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <vector>

#include "sq_common.h"

namespace sq {

constexpr int kPage = SQ_KV_PAGE;  // positions of a page

// Bytes from the start of a (page, head)'s keys / values to one element.
__host__ __device__ inline int kv_k_off(int tok, int dim, int head_dim) {
    return ((((tok >> 4) * (head_dim >> 6) + (dim >> 6)) * 64 + ((dim >> 4) & 3) * 16 + (tok & 15)) << 4) + (dim & 15);
}
__host__ __device__ inline int kv_v_off(int tok, int dim) {
    const int pos = ((tok & 15) << 2) + (tok >> 4);
    return (((dim >> 4) * 64 + (pos >> 4) * 16 + (dim & 15)) << 4) + (pos & 15);
}

// One layer of a pool, by value to the kernels.  Page p of head h: bytes at
// ((p * kv_heads + h) * 2) * 64 * head_dim, scales at p * kv_heads + h.
struct KvView {
    uint8_t* bytes;
    float2* scales;  // (keys', values')
    int kv_heads;
    int head_dim;
};

struct KvSeq {
    int past;    // positions before the step
    int n_new;   // of the step
    int row0;    // its first row in the batch
    int table0;  // its first page in the plan's page list
};
// The new rows of one page: rows row0 .. row0 + n - 1 of the batch go to its
// positions tok0 .. tok0 + n - 1.
struct KvItem {
    int page, row0, tok0, n;
};

struct KvPlanView {
    const KvSeq* seqs;
    const int* pages;
    const KvItem* items;
    const double2* rope;   // [rows][half] (cos, sin), null: nothing is rotated
    const float2* rope32;  // the same in f32: queries, which no integer is decided by
    int n_seqs, n_items, rows, half;
};

// ---- k_kv.hip
int launch_kv_rope(hipStream_t s, const KvPlanView& p, const float* inv_freq, int rows, double2* out, float2* out32);
int launch_kv_append(hipStream_t s, const KvView& kv, const KvPlanView& p, const float* k, size_t k_stride,
                     const float* v, size_t v_stride, uint32_t* bad);
// max_pages: the most pages that a sequence's last `last` positions lie in.
int launch_kv_read(hipStream_t s, const KvView& kv, const KvPlanView& p, int last, int max_pages, float* k_out,
                   float* v_out);

// ---- k_paged.hip
struct PagedArgs {
    const float* q;
    size_t q_stride;
    float* out;
    size_t out_stride;
    int heads, window, sinks;
};
// (on the null stream, with a workspace from the scratch pool)
int launch_sdpa_paged(const std::vector<KvSeq>& seqs, const KvView& kv, const KvPlanView& p, const PagedArgs& a);

}  // namespace sq

struct sq_kv_pool {
    int device = 0;
    size_t n_layers = 0, n_pages = 0, kv_heads = 0, head_dim = 0, half = 0;
    uint8_t* bytes = nullptr;
    float2* scales = nullptr;
    float* inv_freq = nullptr;
};

struct sq_kv_plan {
    const sq_kv_pool* pool = nullptr;
    std::vector<sq::KvSeq> seqs;
    size_t rows = 0, n_items = 0;
    uint8_t* dev = nullptr;  // seqs, items, pages
    size_t dev_size = 0;
    size_t off_items = 0, off_pages = 0;
    double2* rope = nullptr;  // [rows][half], then the same in f32; made by the first call that rotates
    size_t rope_size = 0;
    bool rope_ready = false;
    uint32_t* bad = nullptr;  // pinned: set by a kernel that met a value which is not finite
};

namespace sq {

int kv_pool_create(size_t n_layers, size_t n_pages, size_t kv_heads, size_t head_dim, const float* inv_freq,
                   size_t half, sq_kv_pool** out);
void kv_pool_destroy(sq_kv_pool* p);
int kv_plan_create(const sq_kv_pool* pool, sq_kv_plan** out);
int kv_plan_fill(sq_kv_plan* plan, size_t n_seqs, const uint32_t* past, const uint32_t* n_new, const uint32_t* tables,
                 size_t table_stride);
void kv_plan_destroy(sq_kv_plan* plan);
// What an operator call on a plan checks first, and its views.
int kv_views(sq_kv_plan* plan, size_t layer, bool rotate, const char* what, KvView* kv, KvPlanView* pv);

}  // namespace sq
