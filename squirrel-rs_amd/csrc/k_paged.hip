// Attention over the paged 8-bit key/value cache (kv.h).
//
// Row r of the batch, at position p of its sequence, head h of KV head
// h / (heads / kv_heads):  o = sum_j softmax_j(q . k_j / sqrt(d)) v_j  over the
// positions j <= p, with a window only those with j > p - window or
// j < sinks.
#include <algorithm>
#include <cmath>

#include "kv.h"
#include "scratch.h"

namespace sq {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

inline int check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return set_error(SQ_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
    return 0;
}

// Division of x < 2^31 by a number that a launch knows: with m = ceil(2^32 / d)
// floor(x m / 2^32) is the quotient or one more.  (With the dozen divisions of a
// workgroup's start as the compiler makes them a token over 300 positions took
// 7.3 us instead of 5.7.)
struct alignas(8) Div {
    uint32_t d, m;  // (m = 0: d = 1)
    Div() = default;
    explicit Div(int n) : d((uint32_t)n), m((uint32_t)((((uint64_t)1 << 32) + d - 1) / d)) {}
    __host__ __device__ int operator()(int x) const {
        if (d == 1) return x;
        const uint32_t q = (uint32_t)(((uint64_t)(uint32_t)x * m) >> 32);
        return (int)(q * d > (uint32_t)x ? q - 1 : q);
    }
};

// The query rows of one KV head of a sequence are its n_new * G (position,
// head) pairs, row r = i * G + (head in the group).
//
// The pages that the rows of a tile see, as one list: first those of the
// sinks, then those from the first page of the tile's windows to its last
// position's.
struct Span {
    int sink_pages, first, count;
    __host__ __device__ int page(int i) const { return i < sink_pages ? i : first + i - sink_pages; }
};
__host__ __device__ inline Span tile_span(int pos_lo, int pos_hi, int window, int sinks) {
    Span s{0, 0, pos_hi / kPage + 1};
    if (window > 0 && pos_lo >= window) {
        s.first = (pos_lo - window + 1) / kPage;
        s.sink_pages = (sinks + kPage - 1) / kPage;
        if (s.sink_pages > s.first) s.sink_pages = s.first;
        s.count = s.sink_pages + pos_hi / kPage - s.first + 1;
    }
    return s;
}

// What a launch covers: the sequences with rows_lo <= n_new * G <= rows_hi,
// their pages cut into parts of `chunk` (the last one holds between a half and
// one and a half of it).  The parts' sums stand in the workspace at slot
// (table0 / chunk + sequence + part): a sequence has at most pages / chunk + 1
// parts, so slots do not overlap.
struct Cut {
    int rows_lo, rows_hi, chunk, tiles, splits, pad;
    Div by_chunk, by_group, by_heads;  // chunk, heads / kv_heads, kv_heads
    float* ws;
    __host__ __device__ int parts(int count) const { return count < chunk ? 1 : by_chunk(count + (chunk >> 1)); }
    __host__ __device__ size_t slot(const KvSeq& s, int seq, int part) const {
        return (size_t)by_chunk(s.table0) + seq + part;
    }
};

// Eight stored bytes as f16, exactly: 0x64uu is 1024 + u, u = q + 128.
__device__ __forceinline__ v8h unpack8(uint32_t a, uint32_t b) {
    const uint32_t w[4] = {
        __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u),
        __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)};
    v8h r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const v2h x = __builtin_bit_cast(v2h, w[i]) - (v2h){(_Float16)1152.0f, (_Float16)1152.0f};
        r[2 * i] = x[0], r[2 * i + 1] = x[1];
    }
    return r;
}

// Maximum / sum over the four lanes that share a query (l % 16).
__device__ __forceinline__ float groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float groups_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// Scales of a sequence's pages are taken relative to its first page's (1 where
// that holds zeros), within 2^96 of it either way: their quotients stay in f32.
// A page of zeros may have any scale.
__device__ __forceinline__ float first_unit(float scale) {
    return scale > 0.0f ? fminf(fmaxf(scale, 0x1p-30f), 0x1p30f) : 1.0f;
}
__device__ __forceinline__ float page_unit(float scale, float unit) {
    return scale > 0.0f ? fminf(fmaxf(scale, unit * 0x1p-96f), unit * 0x1p96f) : unit;
}

// E consecutive dimensions of one query row from `d`, rotated; false where one
// is not finite.
template <int E>
__device__ __forceinline__ bool load_query(const float* q, bool vec, const float2* rope, int half, int d, float* x) {
    if (vec) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 f = *(const float4*)(q + d + e);
            x[e] = f.x, x[e + 1] = f.y, x[e + 2] = f.z, x[e + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = q[d + e];
    }
    bool ok = true;
#pragma unroll
    for (int e = 0; e < E; e++) ok = ok && fabsf(x[e]) < INFINITY;
    if (rope && d / 2 < half) {
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const int j = (d + e) / 2;
            const float2 cs = rope[min(j, half - 1)];
            const float u = x[e], v = x[e + 1];
            if (j < half) {
                x[e] = u * cs.x - v * cs.y;
                x[e + 1] = u * cs.y + v * cs.x;
            }
        }
    }
    return ok;
}

// The power of two that brings a row's largest magnitude to 2^13 .. 2^14, and what
// turns products of the scaled row into scores.  A row that is not finite, or
// leaves f32 by its rotation, has NaN scores (shift -1000: its halves are zeros).
__device__ __forceinline__ int query_shift(float amax, float scale, float& cq) {
    if (!(amax < INFINITY)) {
        cq = NAN;
        return -1000;
    }
    const int shift = min(140 - (int)((__builtin_bit_cast(uint32_t, amax) >> 23) & 255), 100);
    cq = ldexpf(scale, -shift);
    return shift;
}
__device__ __forceinline__ void halves(float x, int shift, _Float16& h, _Float16& lo) {
    const float y = shift == -1000 ? 0.0f : ldexpf(x, shift);
    h = (_Float16)y;
    lo = (_Float16)(y - (float)h);
}

// Scores are formed transposed, K Q^T, so that a lane holds one query's
// probabilities of sixteen positions, in the order of the stored values: they
// are the second product's operand as they stand (V^T P^T), and its results,
// dimensions of the same query, are scaled lane by lane.
//
// The cached integers are exact in f16.  A query's elements, scaled by a power
// of two to at most 2^14, and a page's probabilities, times 2^kBase, are split into
// two f16 halves each (x = hi + lo to 2^-22 of x): two products on the matrix
// pipe give what one in f32 would, four times as fast.
//
// A weight w_j = 2^(score_j) comes with its page's value scale: the second
// product's operand is w_j v_scale and the sum of weights takes w_j v_scale *
// (unit / v_scale) in f32.  So the matrix pipe adds to the sums in place, and it is
// the products that count, not the weights, that keep their 22 bits.
// A row's maximum (of score + log2 v_scale) follows in steps: as long as they
// stay within kHeadroom of it nothing is rescaled, and the operands stay below
// 2^(kBase + kHeadroom), in f16's range with kBase bits of room for small ones.
//
// PAGES: the wavefronts take pages in turn for the same 16 rows and meet in LDS;
// otherwise each has its own 16 rows and all walk the same pages.  (32 rows a
// wavefront leave two of them a SIMD: 73 us instead of 55 for 1531 rows.)
//
// What bounds them.  By pages: the reads of the cache, from about 32 pages a
// sequence on (256 sequences and heads of 4096 positions: 134 MB in 24 us, 5.6
// TB/s; 131000 positions of one: 25 us); below that the chain from the launch's
// arguments to a page's bytes and the meeting in LDS, 6 us (300 positions).  By
// rows: the VALU's softmax and halves beside the matrix pipe, 443 TFLOP/s for
// 8192 rows of 32 heads of 64 (two f16 products for one of f32: 577 at the rate
// of a large f16 product), and about 12 us of start and end: 50 us for 1531
// rows behind 517.
constexpr int kStat = 4;  // floats behind a part's sums: the maximum, the sum of weights, the unit, none
constexpr float kBase = 8.0f, kHeadroom = 6.0f;
template <int HD, int NW, bool PAGES>
__global__ __launch_bounds__(NW * 64, HD != 64 ? 2 : PAGES ? 3 : 4) void sdpa_paged_kernel(KvView kv, KvPlanView pl,
                                                                                          PagedArgs a, Cut cut,
                                                                                          float scale) {
    constexpr int C = HD / 64, DT = HD / 16, TR = PAGES ? 16 : NW * 16;
    __shared__ __attribute__((aligned(16))) float s_o[PAGES ? NW * 16 * (HD + 4) : 1];
    __shared__ __attribute__((aligned(16))) _Float16 s_q[2][PAGES ? 16 * HD : 8];
    __shared__ float s_cq[PAGES ? 16 : 1];
    __shared__ __attribute__((aligned(16))) v8h s_kv[PAGES ? 1 : 2][PAGES ? 1 : 16 * C * 64];
    __shared__ float s_m[PAGES ? NW * 16 : 1], s_l[PAGES ? NW * 16 : 1];
    // (heads next to each other: with eight of them each is one XCD's, and a
    // head's tiles share that XCD's L2.  A sequence's last tiles, which see the most
    // pages, come first)
    const int at = cut.by_heads(blockIdx.x), head = blockIdx.x - at * kv.kv_heads, tile = cut.tiles - 1 - at;
    const int part = blockIdx.y, seq = blockIdx.z;
    const KvSeq s = pl.seqs[seq];
    const int G = (int)cut.by_group.d, rows = s.n_new * G;
    if (rows < cut.rows_lo || rows > cut.rows_hi || tile * TR >= rows) return;
    const int row_end = min(rows, (tile + 1) * TR);
    const Span span =
        tile_span(s.past + cut.by_group(tile * TR), s.past + cut.by_group(row_end - 1), a.window, a.sinks);
    const int parts = cut.parts(span.count);
    if (part >= parts) return;
    const int i_end = part == parts - 1 ? span.count : (part + 1) * cut.chunk;
    const bool whole = parts == 1;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, q16 = lane & 15, g = lane >> 4;
    const int row0 = tile * TR + (PAGES ? 0 : wave * 16);  // the wavefront's first row

    // A page's bytes are 8 C pieces of 1 KB, one load of a wavefront each: keys,
    // then values.
    // PAGES: the wavefront's page in registers; the next one's keys are requested
    // before the second product, its values behind it.
    // Otherwise the wavefronts share the work on a page: each loads and unpacks
    // its pieces of the page after next into one of two f16 images in LDS.
    // (Unpacked by every wavefront for itself that is 128 of 286 VALU
    // instructions for 16 rows of a page: 62 us instead of 55 for 1531 rows.)
    constexpr int P = 8 * C, OWN = PAGES ? P : P / NW;
    static_assert(PAGES || P % NW == 0, "whole pieces a wavefront");
    const int step = PAGES ? NW : 1;
    int i = part * cut.chunk + (PAGES ? wave : 0);
    uint4 w[OWN];
    float2 sc = make_float2(0.0f, 0.0f), sc_next = sc;
    const uint4* kb = nullptr;
    // (a page's number is asked for an iteration before its bytes)
    auto number = [&](int i) { return pl.pages[s.table0 + span.page(min(i, i_end - 1))]; };
    auto locate = [&](int id) {
        const size_t cell = (size_t)id * kv.kv_heads + head;
        sc_next = kv.scales[cell];
        kb = (const uint4*)(kv.bytes + cell * 2 * kPage * HD) + lane + (PAGES ? 0 : wave * OWN * 64);
    };
    auto load = [&](int from, int to) {
#pragma unroll
        for (int e = from; e < to; e++) w[e] = kb[e * 64];
    };
    auto share = [&](int buffer) {
#pragma unroll
        for (int e = 0; e < OWN; e++) {
            v8h* to = &s_kv[buffer][((wave * OWN + e) * 2) * 64 + lane];
            to[0] = unpack8(w[e].x, w[e].y);
            to[64] = unpack8(w[e].z, w[e].w);
        }
    };
    const int id0 = number(i);
    int id = number(i + step);
    if (i < i_end) {
        locate(id0);
        load(0, OWN);
    }

    const float unit = first_unit(kv.scales[(size_t)pl.pages[s.table0] * kv.kv_heads + head].y);

    // Queries: [chunk of 64][half of a lane's 16 dimensions].
    v8h qh[C][2], ql[C][2];
    float cq;
    const bool vec = (((uintptr_t)a.q | (a.q_stride * 4)) & 15) == 0;
    auto query = [&](int r) {
        const int i = cut.by_group(r);
        return a.q + ((size_t)s.row0 + i) * a.q_stride + (size_t)(head * G + r - i * G) * HD;
    };
    auto rope = [&](int r) { return pl.rope32 ? pl.rope32 + ((size_t)s.row0 + cut.by_group(r)) * pl.half : nullptr; };
    const int own = min(row0 + q16, rows - 1);  // the lane's row
    const int pos = s.past + cut.by_group(own), w0 = a.window && a.window <= pos ? pos - a.window + 1 : 0;
    if constexpr (PAGES) {
        // Once for the workgroup, HD / 16 consecutive dimensions a thread (16 lanes
        // are a row), handed over in the operand's order.  (By every wavefront for
        // itself a load's 64 lanes are in as many cache lines: 33 us instead of 28
        // for 48 chats.)
        constexpr int E = HD / 16;
        static_assert(NW >= 4, "a thread has one piece of the rows");
        if (threadIdx.x < 256) {
            const int e0 = (threadIdx.x & 15) * E, k = threadIdx.x >> 4, r = row0 + k;
            float x[E] = {};
            float amax = 0.0f, c = 0.0f;
            bool ok = true;
            if (r < rows) {
                ok = load_query<E>(query(r), vec, rope(r), pl.half, e0, x);
#pragma unroll
                for (int e = 0; e < E; e++) amax = fmaxf(amax, fabsf(x[e]));
            }
            const int shift = query_shift(sq_row_max(ok ? amax : INFINITY), scale, c);
            if ((threadIdx.x & 15) == 0) s_cq[k] = c;
            // dimension d: chunk d / 64, lane group (d / 16) % 4, half (d / 8) % 2
            const int at = (((e0 >> 6) * 2 + ((e0 >> 3) & 1)) * 64 + ((e0 >> 4) & 3) * 16 + k) * 8 + (e0 & 7);
#pragma unroll
            for (int e = 0; e < E; e++) halves(x[e], shift, s_q[0][at + e], s_q[1][at + e]);
        }
        __syncthreads();
        cq = s_cq[q16];
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                qh[c][h] = *(const v8h*)&s_q[0][((c * 2 + h) * 64 + lane) * 8];
                ql[c][h] = *(const v8h*)&s_q[1][((c * 2 + h) * 64 + lane) * 8];
            }
    } else {
        float x[C][16];
        float amax = 0.0f;
        bool ok = true;
#pragma unroll
        for (int c = 0; c < C; c++) {
            ok = load_query<16>(query(own), vec, rope(own), pl.half, 64 * c + 16 * g, x[c]) && ok;
#pragma unroll
            for (int e = 0; e < 16; e++) amax = fmaxf(amax, fabsf(x[c][e]));
        }
        const int shift = query_shift(groups_max(ok ? amax : INFINITY), scale, cq);
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                _Float16 h, lo;
                halves(x[c][e], shift, h, lo);
                qh[c][e / 8][e % 8] = h, ql[c][e / 8][e % 8] = lo;
            }
    }

    // (-1 that the compiler does not know to be: p - h then takes the f16 half as it
    // is, where it would convert it to f32 first)
    float minus = -1.0f;
    asm volatile("" : "+v"(minus));
    v4f o[DT];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // rows between the tile's first and last position see a page whole where both do
    const int pos_lo = s.past + cut.by_group(row0), pos_hi = s.past + cut.by_group(min(rows, row0 + 16) - 1);
    const int w0_hi = a.window && a.window <= pos_hi ? pos_hi - a.window + 1 : 0;

    int turn = 0;
    if constexpr (!PAGES) {  // (a launch's parts are never empty)
        share(0);
        sc = sc_next;
        if (i + 1 < i_end) {
            locate(id);
            load(0, OWN);
            id = number(i + 2);
        }
        __syncthreads();
    }
    for (; i < i_end; i += step) {
        const int page = span.page(i);
        const bool more = i + step < i_end;
        if constexpr (PAGES) {
            sc = sc_next;
        } else if (more) {
            share(turn ^ 1);
        }
        // half h of piece e
        auto half = [&](int e, int h) {
            if constexpr (PAGES)
                return h ? unpack8(w[e].z, w[e].w) : unpack8(w[e].x, w[e].y);
            else
                return s_kv[turn][(e * 2 + h) * 64 + lane];
        };
        // scores [tile of 16 positions][position 4 g + r]
        v4f x[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            x[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < C; c++) {
                const v8h k0 = half(t * C + c, 0), k1 = half(t * C + c, 1);
                x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[c][0], x[t], 0, 0, 0);
                x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[c][1], x[t], 0, 0, 0);
                x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[c][0], x[t], 0, 0, 0);
                x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[c][1], x[t], 0, 0, 0);
            }
        }
        const bool full = (page + 1) * kPage - 1 <= pos_lo && (page * kPage >= w0_hi || (page + 1) * kPage <= a.sinks);
        const float vs = page_unit(sc.y, unit), lr = __builtin_amdgcn_logf(vs), back = unit / vs;
        float cs = cq * sc.x;
        if (!full) {
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int at = page * kPage + 16 * t + 4 * g + r;
                    const bool hidden = (at > pos) | ((at < w0) & (at >= a.sinks));
                    x[t][r] = hidden ? -INFINITY : x[t][r] * cs;
                }
            cs = 1.0f;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) mx = fmaxf(mx, x[t][r]);
        mx = mx * cs + lr;
        if (__any(mx > m + kHeadroom)) {
            const float mn = fmaxf(m, groups_max(mx));
            const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= alpha;
        }
        const float off = kBase - (m == -INFINITY ? 0.0f : m) + lr;
        float sum = 0.0f;
        v8h ph[2], plo[2];
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int t = 0; t < 4; t += 2) {
                const v2f p = {__builtin_amdgcn_exp2f(fmaf(x[t][r], cs, off)),
                               __builtin_amdgcn_exp2f(fmaf(x[t + 1][r], cs, off))};
                sum += p[0] + p[1];
                const v2h h = __builtin_convertvector(p, v2h);
                const v2f rest = {fmaf((float)h[0], minus, p[0]), fmaf((float)h[1], minus, p[1])};
                const v2h w = __builtin_convertvector(rest, v2h);
                const int j = 4 * r + t;
                ph[j / 8][j % 8] = h[0], ph[j / 8][j % 8 + 1] = h[1];
                plo[j / 8][j % 8] = w[0], plo[j / 8][j % 8 + 1] = w[1];
            }
        l += sum * back;
        if (PAGES && more) {
            locate(id);
            load(0, 4 * C);
            id = number(i + 2 * step);
        }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const v8h v0 = half(4 * C + d, 0), v1 = half(4 * C + d, 1);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, plo[0], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, plo[1], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0], o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[1], o[d], 0, 0, 0);
        }
        if constexpr (PAGES) {
            if (more) load(4 * C, P);
        } else {
            sc = sc_next;
            if (i + 2 < i_end) {
                locate(id);
                load(0, OWN);
                id = number(i + 3);
            }
            turn ^= 1;
            __syncthreads();
        }
    }
    l = groups_sum(l);

    // where four of row r's sums go: its output, or its part of the workspace
    const bool vec_out = (((uintptr_t)a.out | (a.out_stride * 4)) & 15) == 0;
    auto emit = [&](int r, int d, v4f v, float mm, float ll) {
        if (whole) {
            const int i = cut.by_group(r);
            float* out = a.out + ((size_t)s.row0 + i) * a.out_stride + (size_t)(head * G + r - i * G) * HD + d;
            v *= unit / ll;
            if (vec_out) {
                *(v4f*)out = v;
            } else {
#pragma unroll
                for (int k = 0; k < 4; k++) out[k] = v[k];
            }
        } else {
            const size_t at = (cut.slot(s, seq, part) * kv.kv_heads + head) * cut.rows_hi + r;
            float* w = cut.ws + at * (HD + kStat);
            *(v4f*)(w + d) = v;
            if (d == 0) *(v4f*)(w + HD) = v4f{mm, ll, unit, 0.0f};
        }
    };
    if constexpr (PAGES) {
        // (a wavefront that saw nothing has no weight; NaN scores keep their NaN)
        if (row0 + q16 < rows) {
            const int k = wave * 16 + q16;
            if (g == 0) s_m[k] = m, s_l[k] = l;
#pragma unroll
            for (int d = 0; d < DT; d++) *(v4f*)&s_o[k * (HD + 4) + 16 * d + 4 * g] = o[d];
        }
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * (HD / 4); e += NW * 64) {
            const int r = e / (HD / 4), d = e % (HD / 4) * 4;
            if (row0 + r >= rows) break;
            float mm = -INFINITY, ll = 0.0f;
            v4f v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < NW; w++) mm = fmaxf(mm, s_m[w * 16 + r]);
            const float base = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const int k = w * 16 + r;
                const float m1 = s_m[k], l1 = s_l[k];
                const float f = __builtin_amdgcn_exp2f((m1 == -INFINITY && l1 != 0.0f ? 0.0f : m1) - base);
                ll += l1 * f;
                v += *(const v4f*)&s_o[k * (HD + 4) + d] * f;
            }
            emit(row0 + r, d, v, mm, ll);
        }
    } else if (row0 + q16 < rows) {
#pragma unroll
        for (int d = 0; d < DT; d++) emit(own, 16 * d + 4 * g, o[d], m, l);
    }
}

// The parts of the rows whose pages were cut, from (sequence, KV head, row).
// W wavefronts share a row: all four of a workgroup where rows are few and parts
// many (131000 positions: 32 rows of 93 parts, 5 us), one where it is the other way.
// The lanes find the factors of 64 parts, then a wavefront adds every W-th
// part, eight in flight at a time.
template <int HD, int W>
__global__ __launch_bounds__(256) void sdpa_merge_kernel(KvView kv, KvPlanView pl, PagedArgs a, Cut cut,
                                                         int tile_rows) {
    constexpr int C = HD / 64, IN = 8;
    __shared__ float s_o[4][HD];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, mine = wave % W;
    const int seq = blockIdx.y, at = cut.by_heads(blockIdx.x), head = blockIdx.x - at * kv.kv_heads;
    const int r = at * (4 / W) + wave / W;
    const KvSeq s = pl.seqs[seq];
    const int G = (int)cut.by_group.d, rows = s.n_new * G;
    int parts = 1;
    if (rows >= cut.rows_lo && rows <= cut.rows_hi && r < rows) {
        const int tile = r / tile_rows, row_end = min(rows, (tile + 1) * tile_rows);
        const Span span =
            tile_span(s.past + cut.by_group(tile * tile_rows), s.past + cut.by_group(row_end - 1), a.window, a.sinks);
        parts = cut.parts(span.count);
    }
    if (parts == 1) return;  // (W = 4: the whole workgroup)
    const size_t stride = (size_t)kv.kv_heads * cut.rows_hi * (HD + kStat);
    const float* w = cut.ws + ((cut.slot(s, seq, 0) * kv.kv_heads + head) * cut.rows_hi + r) * (HD + kStat);
    // part i's maximum, sum of weights and unit; its sums and those of the next IN - 1
    // that are this wavefront's
    auto stat = [&](int i) {
        return i < parts ? *(const v4f*)(w + i * stride + HD) : v4f{-INFINITY, 0.0f, 0.0f, 0.0f};
    };
    float v[IN][C];
    auto sums = [&](int i, int end) {
#pragma unroll
        for (int j = 0; j < IN; j++)
#pragma unroll
            for (int c = 0; c < C; c++)
                v[j][c] = i + W * j < end ? w[(i + W * j) * stride + 64 * c + lane] : 0.0f;
    };
    v4f st = stat(lane);
    const float mine_unit = st[2];  // (a bit cast of a vector's element would take its first)
    const float unit = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, mine_unit), 0));
    sums(mine, min(parts, 64));  // (in flight while the factors form)
    float mm = st[0], ll = 0.0f, o[C] = {};
    for (int i = lane + 64; i < parts; i += 64) mm = fmaxf(mm, stat(i)[0]);
    mm = sq_wave_max(mm);
    for (int i0 = 0; i0 < parts; i0 += 64) {
        if (i0) st = stat(i0 + lane);
        // (a part that saw nothing adds nothing; NaN scores keep their NaN)
        const float f = __builtin_amdgcn_exp2f((st[0] == -INFINITY && st[1] != 0.0f ? 0.0f : st[0]) -
                                               (mm == -INFINITY ? 0.0f : mm));
        ll += st[1] * f;
        const int n = min(parts - i0, 64);
        for (int k = mine; k < n; k += W * IN) {
            if (i0 + k != mine) sums(i0 + k, i0 + n);
#pragma unroll
            for (int j = 0; j < IN; j++) {
                const float fj = __builtin_bit_cast(
                    float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(k + W * j, 63)));
                if (k + W * j < n)
#pragma unroll
                    for (int c = 0; c < C; c++) o[c] += v[j][c] * fj;
            }
        }
    }
    ll = sq_wave_sum(ll);
    if constexpr (W > 1) {
#pragma unroll
        for (int c = 0; c < C; c++) s_o[wave][64 * c + lane] = o[c];
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int d = 64 * c + lane;
            o[c] = (s_o[0][d] + s_o[1][d]) + (s_o[2][d] + s_o[3][d]);
        }
    }
    const int i = cut.by_group(r);
    float* out = a.out + ((size_t)s.row0 + i) * a.out_stride + (size_t)(head * G + r - i * G) * HD;
#pragma unroll
    for (int c = 0; c < C; c++) out[64 * c + lane] = o[c] * (unit / ll);
}

// Sequences of few rows: wavefronts over pages, tiles of 16 rows, which read
// the pages once each (from the L2 after the first).  More rows: wavefronts over
// rows, tiles of 64, a page unpacked once for all of them.  Measured on 32
// sequences of 8 KV heads, 64 dimensions, 512 / 4096 positions (us): 40 rows 11 /
// 47 by pages and 15 / 86 by rows, 96 rows 19 / 83 and 19 / 104, 128 rows 23 /
// 107 and 19 / 102; with 128 dimensions 96 rows 33 / 158 and 29 / 166.
constexpr int kFewWaves = 4, kFewRows = 96, kTileFew = 16, kTileMany = 64;
// Pages are cut into parts until the launch has about so many workgroups (three
// a CU by pages; fewer and 48 chats of up to 8000 positions take 25 us instead
// of 22), of at least 16 pages by pages (four a wavefront) and 8 by rows.  Tiles
// of rows that are half as many as the target already are not cut: the merge's
// traffic costs more than the idle CUs (1024 rows behind 8192: 205 us uncut,
// 185 + 19 in two parts).
constexpr int kTarget = 768, kTargetMany = 512;

struct Launch {
    Cut cut;
    size_t floats;
    bool any;
};
Launch plan_launch(const std::vector<KvSeq>& seqs, const KvView& kv, const PagedArgs& a, bool many) {
    const int G = a.heads / kv.kv_heads, tile = !many ? kTileFew : kTileMany;
    Launch r{};
    r.cut.rows_lo = many ? kFewRows + 1 : 1;
    r.cut.by_group = Div(G);
    r.cut.by_heads = Div(kv.kv_heads);
    long long work = 0, groups = 0, pages = 0;
    int longest = 0;
    for (const KvSeq& s : seqs) {
        const int rows = s.n_new * G;
        pages = s.table0 + (s.past + s.n_new + kPage - 1) / kPage;
        if (rows < 1 || (rows > kFewRows) != many) continue;
        r.any = true;
        const int tiles = (rows + tile - 1) / tile;
        r.cut.rows_hi = std::max(r.cut.rows_hi, rows);
        r.cut.tiles = std::max(r.cut.tiles, tiles);
        groups += tiles;
        for (int t = 0; t < tiles; t++) {
            const Span sp = tile_span(s.past + t * tile / G, s.past + (std::min(rows, (t + 1) * tile) - 1) / G,
                                      a.window, a.sinks);
            work += sp.count;
            longest = std::max(longest, sp.count);
        }
    }
    work *= kv.kv_heads;
    groups *= kv.kv_heads;
    const int least = many ? 8 : 4 * kFewWaves;
    const int target = many ? kTargetMany : kTarget;
    long long chunk = std::max<long long>(least, (work + target - 1) / target);
    if (many && groups >= target / 2) chunk = 2ll * longest;
    for (;; chunk *= 2) {
        r.cut.chunk = (int)std::min<long long>(chunk, 2ll * longest + 1);
        r.cut.by_chunk = Div(r.cut.chunk);
        r.cut.splits = r.cut.parts(longest);
        r.floats = r.cut.splits < 2 ? 0
                                    : (size_t)(pages / r.cut.chunk + seqs.size() + 1) * kv.kv_heads * r.cut.rows_hi *
                                          (kv.head_dim + kStat);
        if (r.floats <= ((size_t)64 << 20)) break;  // 256 MB
    }
    return r;
}

template <int HD, int NW, bool PAGES>
int launch_one(const Launch& l, const KvView& kv, const KvPlanView& p, const PagedArgs& a) {
    const float scale = 1.4426950408889634f / sqrtf((float)HD);  // scores in units of log 2
    const size_t grid = (size_t)l.cut.tiles * kv.kv_heads;
    constexpr int W = PAGES ? 4 : 1;  // wavefronts that share a row of the merge
    const size_t merge = (size_t)(l.cut.rows_hi * W + 3) / 4 * kv.kv_heads;
    if (!grid_fits(grid, NW * 64) || !grid_fits(merge, 256))
        return set_error(SQ_ERR_SHAPE, "sdpa_paged: ShapeMismatch (too many rows)");
    hipLaunchKernelGGL((sdpa_paged_kernel<HD, NW, PAGES>), dim3((unsigned)grid, l.cut.splits, p.n_seqs),
                       dim3(NW * 64), 0, nullptr, kv, p, a, l.cut, scale);
    if (l.cut.splits > 1)
        hipLaunchKernelGGL((sdpa_merge_kernel<HD, W>), dim3((unsigned)merge, p.n_seqs), dim3(256), 0, nullptr, kv, p, a,
                           l.cut, PAGES ? 16 : NW * 16);
    return check_launch("sdpa_paged");
}

}  // namespace

int launch_sdpa_paged(const std::vector<KvSeq>& seqs, const KvView& kv, const KvPlanView& p, const PagedArgs& a) {
    Launch l[2] = {plan_launch(seqs, kv, a, false), plan_launch(seqs, kv, a, true)};
    Tmp ws;  // (the second launch follows the first's merge)
    const size_t floats = std::max(l[0].floats, l[1].floats);
    int st = 0;
    if (floats && (st = ws.alloc(floats * sizeof(float)))) return st;
    for (int many = 0; many < 2 && !st; many++) {
        if (!l[many].any) continue;
        l[many].cut.ws = (float*)ws.p;
        if (kv.head_dim == 64)
            st = many ? launch_one<64, 4, false>(l[1], kv, p, a) : launch_one<64, kFewWaves, true>(l[0], kv, p, a);
        else
            st = many ? launch_one<128, 4, false>(l[1], kv, p, a) : launch_one<128, kFewWaves, true>(l[0], kv, p, a);
    }
    return st;
}

}  // namespace sq
