// Page scores and page selection of Quest over a paged cache.
//
//  * score:  sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo with q+ = max(q, 0), q- = min(q, 0):
//    a product of the query heads with pages as rows of 2 head_dim channels, so it runs on the tensor
//    cores (exact 16-bit products, fp32 sums).  Bound by reading the bounds once: 8 sequences of
//    8192 pages, 8 KV heads of 128, 277 MB with the scores in 46 us (6.0 TB/s).
//  * select: one CTA per query head holds the row's order keys in registers and finds the key
//    of rank budget - 1 by histograms of 2048 bins over the range that is left: first the row's own
//    [least, largest], which spreads the keys over the bins whatever their exponents are, then the
//    bin that holds the rank, until that bin is taken whole (two rounds as a rule, three at most).  The picks are
//    written as a bitmap; the last query head of a KV head merges its group's bitmaps into an
//    ascending page list with head masks.  Latency-bound: 8.5 us for 32 rows of 2048 pages, of
//    which the launch is 3, the keys' arrival 1.5, the search 2 and ticket and merge 2 (7.3 us in a CUDA
//    graph); 256 rows of 8192 pages 17 us.
#include <cmath>
#include <type_traits>

#include "key_range.h"
#include "paged_core.cuh"

namespace popkv {
namespace {

constexpr int kScoreThreads = 128;
constexpr uint32_t kFull = 0xffffffffu;
constexpr int64_t kTicketBytes = POPKV_PAGED_TICKET_BYTES;
constexpr int64_t kMaxItems = kTicketBytes / 4 - 1;

// ------------------------------------------------------------------------ score
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Halves of a packed 16-bit pair that are negative (NEG) or not, the others cleared.  A NaN
// stays where its sign puts it.
template <bool NEG>
__device__ __forceinline__ uint32_t part_of(uint32_t w) {
    const uint32_t neg = ((w >> 15) & 0x00010001u) * 0xffffu;  // 0xffff in negative halves
    return w & (NEG ? neg : ~neg);
}

struct ScoreArgs {
    const void* q;
    const void* bounds;
    int64_t pages;
    const int32_t* table;
    int64_t table_stride;
    int width;
    const int32_t* lengths;
    int q_heads, kv_heads, G, head_dim, page_size;
    bool q_vec;
    int runs;  // of 8 pages per warp
    float* scores;
};

// A warp walks runs of 8 pages of one (sequence, KV head).  A page's 2 head_dim bounds go straight
// from global memory into B fragments: lane (n, c) holds 16-byte pieces 4 x + c of page n.  The next
// run's bounds, and the table entries of the one after it, are on their way while one is multiplied.
template <typename T, int DP>
__global__ void __launch_bounds__(kScoreThreads, DP <= 128 ? 4 : 2) paged_score_kernel(ScoreArgs a) {
    pdl_wait();
    constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr int kPieces = DP / 32;  // 16-byte pieces per lane, of the smallest and as many of the largest keys
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = lane >> 2, col = lane & 3;
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int first = (blockIdx.x * (kScoreThreads / 32) + warp) * a.runs * 8;
    if (first >= a.width) return;
    const int end = min(a.width, first + a.runs * 8);
    const int64_t len = a.lengths[b];
    const int32_t* columns = a.table + b * a.table_stride;
    auto entry = [&](int c0) {
        const int column = c0 + row;
        return column < end && static_cast<int64_t>(column) * a.page_size < len ? columns[column] : -1;
    };
    auto is_page = [&](int page) { return page >= 0 && page < a.pages; };
    auto fetch = [&](uint4 (&lo)[kPieces], uint4 (&hi)[kPieces], int page) {
        const bool mapped = is_page(page);
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const T*>(a.bounds) +
                                                        (mapped ? static_cast<int64_t>(page) * a.kv_heads + kvh : 0) * 2 * a.head_dim);
#pragma unroll
        for (int x = 0; x < kPieces; ++x) {
            const int piece = 4 * x + col;
            const bool in = mapped && 8 * piece < a.head_dim;
            lo[x] = in ? __ldcs(p + piece) : make_uint4(0u, 0u, 0u, 0u);
            hi[x] = in ? __ldcs(p + a.head_dim / 8 + piece) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    // Queries in the same channel order, as A fragments whose rows 0-7 are q- and rows 8-15 q+ of 8
    // heads: multiplied by lo, rows 0-7 are what is wanted, by hi, rows 8-15.
    uint32_t qf[kPieces][2][4];
    auto load_queries = [&](int g0) {
#pragma unroll
        for (int x = 0; x < kPieces; ++x) {
            const int ch = 8 * (4 * x + col);
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if (g0 + row < a.G && ch < a.head_dim)
                w = load_raw8<T>(static_cast<const T*>(a.q) + (static_cast<int64_t>(b) * a.q_heads + kvh * a.G + g0 + row) * a.head_dim + ch,
                                 a.q_vec);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    qf[x][h][2 * r] = part_of<true>(ws[2 * h + r]);
                    qf[x][h][2 * r + 1] = part_of<false>(ws[2 * h + r]);
                }
        }
    };
    auto score = [&](const uint4 (&lo)[kPieces], const uint4 (&hi)[kPieces], int page, int c0) {
        const uint32_t ok = __ballot_sync(kFull, is_page(page));
        for (int g0 = 0; g0 < a.G; g0 += 8) {
            if (a.G > 8) load_queries(g0);
            float s[2][4] = {};
#pragma unroll
            for (int x = 0; x < kPieces; ++x)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    mma16816<kBf16>(s[0], qf[x][h][0], qf[x][h][1], qf[x][h][2], qf[x][h][3], h ? lo[x].z : lo[x].x, h ? lo[x].w : lo[x].y);
                    mma16816<kBf16>(s[1], qf[x][h][0], qf[x][h][1], qf[x][h][2], qf[x][h][3], h ? hi[x].z : hi[x].x, h ? hi[x].w : hi[x].y);
                }
            // Column 2 col + e was loaded by the lanes of row 2 col + e.
            if (g0 + row < a.G) {
                float* out = a.scores + (static_cast<int64_t>(b) * a.q_heads + kvh * a.G + g0 + row) * a.width + c0 + 2 * col;
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (c0 + 2 * col + e < end) out[e] = (ok >> (8 * col + 4 * e)) & 1u ? s[0][e] + s[1][2 + e] : -INFINITY;
            }
        }
    };
    // Two register buffers take turns.
    int page0 = entry(first), page1 = entry(first + 8);
    uint4 lo0[kPieces], hi0[kPieces], lo1[kPieces], hi1[kPieces];
    fetch(lo0, hi0, page0);
    if (a.G <= 8) load_queries(0);
    for (int c0 = first; c0 < end; c0 += 16) {
        fetch(lo1, hi1, page1);
        const int after0 = entry(c0 + 16);
        score(lo0, hi0, page0, c0);
        page0 = after0;
        fetch(lo0, hi0, page0);
        const int after1 = entry(c0 + 24);
        if (c0 + 8 < end) score(lo1, hi1, page1, c0 + 8);
        page1 = after1;
    }
    pdl_trigger();
}

// ----------------------------------------------------------------------- select
// Larger score, larger key; NaN above everything, -infinity (never selected) is 0.
__device__ __forceinline__ uint32_t select_key(float x) {
    if (x != x) return 0xffffffffu;
    if (x == -INFINITY) return 0u;
    return order_key(x);
}

struct SelectArgs {
    const float* scores;
    int width;
    const int32_t* lengths;
    int q_heads, kv_heads, page_size, budget;
    popkv_page_list list;
    uint32_t* tickets;
    uint32_t* bitmaps;  // [batch * q_heads][words]
    int words;
};

// KPT keys per thread in registers; KPT = 0: rows too long for that are read again (L2) at every step.
template <int NT, int KPT>
__global__ void __launch_bounds__(NT) paged_select_kernel(SelectArgs a) {
    pdl_trigger();
    pdl_wait();
    constexpr int kWarps = NT / 32;
    constexpr int kRounds = KPT > 0 ? KPT : 1;
    constexpr int kBins = 1 << KeyRange::kBits, kPer = kBins / NT;  // bins per thread in the scan
    __shared__ __align__(16) uint32_t s_hist[kBins];
    __shared__ uint32_t s_warp[2][kWarps];
    __shared__ uint32_t s_ties[kRounds * kWarps];
    __shared__ uint32_t s_pick[4];  // bin, keys above it, keys in it; ticket
    __shared__ uint32_t s_first[kBins];  // place of a word's first page in the list
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x, b = row / a.q_heads;
    const int G = a.q_heads / a.kv_heads;
    const float* s = a.scores + static_cast<int64_t>(row) * a.width;
    int64_t len = a.lengths[b];
    len = len < 0 ? 0 : min(len, static_cast<int64_t>(a.width) * a.page_size);
    const int n = len > 0 ? static_cast<int>((len - 1) / a.page_size) : 0;  // older pages; column n is the newest
    const uint32_t want = static_cast<uint32_t>(a.budget - 1);
    uint32_t key[kRounds];
    if constexpr (KPT > 0) {  // every column: the loads need not wait for the length
#pragma unroll
        for (int k = 0; k < KPT; ++k) key[k] = __float_as_uint(k * NT + tid < a.width ? __ldcg(s + k * NT + tid) : 0.0f);
#pragma unroll
        for (int k = 0; k < KPT; ++k) key[k] = k * NT + tid < n ? select_key(__uint_as_float(key[k])) : 0u;
    }
    for (int i = tid; i < kBins; i += NT) s_hist[i] = 0u;
    auto each = [&](auto&& f) {  // every key that may be taken
        if constexpr (KPT > 0) {
#pragma unroll
            for (int k = 0; k < KPT; ++k)
                if (key[k] != 0u) f(key[k]);
        } else {
            for (int i = tid; i < n; i += NT) {
                const uint32_t k = select_key(__ldcg(s + i));
                if (k != 0u) f(k);
            }
        }
    };
    // thr: the least key that is taken, at least 1; take: how many of the keys equal to thr.
    uint32_t thr = 1u, take = 0xffffffffu;
    if (want < static_cast<uint32_t>(n)) {
        uint32_t lo = 0xffffffffu, hi = 0u, count = 0u;
        each([&](uint32_t k) { lo = min(lo, k); hi = max(hi, k); ++count; });
        lo = __reduce_min_sync(kFull, lo);
        hi = __reduce_max_sync(kFull, hi);
        count = __reduce_add_sync(kFull, count);
        if (lane == 0) { s_warp[0][warp] = lo; s_warp[1][warp] = hi; s_ties[warp] = count; }
        __syncthreads();
        lo = __reduce_min_sync(kFull, lane < kWarps ? s_warp[0][lane] : 0xffffffffu);
        hi = __reduce_max_sync(kFull, lane < kWarps ? s_warp[1][lane] : 0u);
        count = __reduce_add_sync(kFull, lane < kWarps ? s_ties[lane] : 0u);
        if (want == 0u) {
            thr = 0xffffffffu;
            take = 0u;
        } else if (want < count) {
            uint32_t left = want;  // rank wanted among the keys of the range
            KeyRange range{lo, hi};
            for (int step = 1;; ++step) {
                const int shift = range.shift();
                each([&](uint32_t k) {
                    if (range.holds(k)) atomicAdd(s_hist + range.bin(k, shift), 1u);
                });
                __syncthreads();
                // Suffix sums: thread t owns bins kPer t ..; keys in the bins above its own.
                uint32_t c[kPer], sum = 0u;
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    c[i] = s_hist[kPer * tid + i];
                    sum += c[i];
                }
                uint32_t incl = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t y = __shfl_down_sync(kFull, incl, o);
                    if (lane + o < 32) incl += y;
                }
                if (lane == 0) s_warp[0][warp] = incl;
                __syncthreads();
                uint32_t above = incl - sum + __reduce_add_sync(kFull, lane > warp && lane < kWarps ? s_warp[0][lane] : 0u);
#pragma unroll
                for (int i = kPer - 1; i >= 0; --i) {
                    if (above < left && above + c[i] >= left) {
                        s_pick[0] = kPer * tid + i;
                        s_pick[1] = above;
                        s_pick[2] = c[i];
                    }
                    above += c[i];
                    s_hist[kPer * tid + i] = 0u;  // for the next round
                }
                __syncthreads();
                range.keep(s_pick[0], shift);
                left -= s_pick[1];
                const bool whole = left == s_pick[2];  // the bin is taken whole
                if (whole || shift == 0 || step == KeyRange::kSteps) {  // the last step's bins hold one key each
                    thr = range.lo;
                    take = whole ? 0xffffffffu : left;
                    break;
                }
                // The next writes of s_warp and s_pick come after two more barriers.
            }
        }
    }
    const bool split = take != 0xffffffffu && take != 0u;  // some of the keys equal to thr are left out
    uint32_t* map = a.bitmaps + static_cast<int64_t>(row) * a.words;
    __syncthreads();
    if constexpr (KPT > 0) {
        if (split) {  // ties go to the lowest columns: rank them
#pragma unroll
            for (int k = 0; k < KPT; ++k) {
                const uint32_t w = __ballot_sync(kFull, key[k] == thr);
                if (lane == 0) s_ties[k * kWarps + warp] = __popc(w);
            }
            __syncthreads();
            if (warp == 0) {
                uint32_t base = 0;
                for (int i = 0; i < KPT * kWarps; i += 32) {
                    const uint32_t c = i + lane < KPT * kWarps ? s_ties[i + lane] : 0u;
                    uint32_t incl = c;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const uint32_t y = __shfl_up_sync(kFull, incl, o);
                        if (lane >= o) incl += y;
                    }
                    if (i + lane < KPT * kWarps) s_ties[i + lane] = base + incl - c;
                    base += __shfl_sync(kFull, incl, 31);
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int k = 0; k < KPT; ++k) {
            const int i = k * NT + tid;
            bool pick = key[k] >= thr && take != 0u;
            if (split) {
                const uint32_t w = __ballot_sync(kFull, key[k] == thr);
                if (key[k] == thr) pick = s_ties[k * kWarps + warp] + __popc(w & ((1u << lane) - 1u)) < take;
            }
            if (i == n && len > 0) pick = true;
            const uint32_t word = __ballot_sync(kFull, pick);
            if (lane == 0 && (i >> 5) < a.words) map[i >> 5] = word;
        }
    } else {
        uint32_t taken = 0;
        for (int base = 0; base < a.words * 32; base += NT) {
            const int i = base + tid;
            const uint32_t k = i < n ? select_key(__ldcg(s + i)) : 0u;
            bool pick = k >= thr && take != 0u;
            if (split) {
                const uint32_t w = __ballot_sync(kFull, k == thr);
                if (lane == 0) s_ties[warp] = __popc(w);
                __syncthreads();
                if (k == thr) {
                    uint32_t before = taken;
                    for (int v = 0; v < warp; ++v) before += s_ties[v];
                    pick = before + __popc(w & ((1u << lane) - 1u)) < take;
                }
                for (int v = 0; v < kWarps; ++v) taken += s_ties[v];
                __syncthreads();
            }
            if (i == n && len > 0) pick = true;
            const uint32_t word = __ballot_sync(kFull, pick);
            if (lane == 0 && (i >> 5) < a.words) map[i >> 5] = word;
        }
    }
    // The last query head of the group merges.  One thread's fences order the block's words
    // (the barriers before and after carry them) with the ticket.
    const int item = row / G;
    __syncthreads();
    if (tid == 0) {
        uint32_t t;  // releases the row's bitmap, acquires those of the others
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(t) : "l"(a.tickets + item) : "memory");
        s_pick[3] = t;
    }
    __syncthreads();
    if (s_pick[3] != static_cast<uint32_t>(G) - 1u) return;
    if (tid == 0) a.tickets[item] = 0u;
    const uint32_t* maps = a.bitmaps + static_cast<int64_t>(item) * G * a.words;
    int32_t* pages = a.list.pages + static_cast<int64_t>(item) * a.list.capacity;
    uint32_t* heads = a.list.heads + static_cast<int64_t>(item) * a.list.capacity;
    // A stretch of words at a time in shared memory: their pages are counted a thread per word, then
    // written a warp per word (32 columns, a lane each).
    const int stretch = min(a.words, kBins / G);
    uint32_t done = 0;
    for (int base = 0; base < a.words; base += stretch) {
        const int here = min(stretch, a.words - base);
        for (int i = tid; i < G * here; i += NT) s_hist[i] = __ldcg(maps + static_cast<int64_t>(i / here) * a.words + base + i % here);
        __syncthreads();
        for (int w0 = 0; w0 < here; w0 += NT) {
            const int w = w0 + tid;
            uint32_t any = 0;
            if (w < here)
                for (int g = 0; g < G; ++g) any |= s_hist[g * here + w];
            uint32_t incl = __popc(any);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(kFull, incl, o);
                if (lane >= o) incl += y;
            }
            if (lane == 31) s_warp[0][warp] = incl;
            __syncthreads();
            const uint32_t sums = lane < kWarps ? s_warp[0][lane] : 0u;
            const uint32_t before = done + __reduce_add_sync(kFull, lane < warp ? sums : 0u);
            if (w < here) s_first[w] = before + incl - __popc(any);
            done += __reduce_add_sync(kFull, sums);
            __syncthreads();
        }
        for (int w = warp; w < here; w += kWarps) {
            uint32_t mask = 0;
            for (int g = 0; g < G; ++g) mask |= ((s_hist[g * here + w] >> lane) & 1u) << g;
            const uint32_t any = __ballot_sync(kFull, mask != 0u);
            const uint32_t at = s_first[w] + __popc(any & ((1u << lane) - 1u));
            if (mask != 0u && at < a.list.capacity) {
                pages[at] = 32 * (base + w) + lane;
                heads[at] = mask;
            }
        }
        __syncthreads();
    }
    const uint32_t total = done;
    if (tid == 0) a.list.counts[item] = static_cast<int32_t>(min(static_cast<int64_t>(total), a.list.capacity));
}

}  // namespace
}  // namespace popkv

using namespace popkv;

extern "C" int popkv_paged_score(const void* q, const popkv_paged_cache* cache, const int32_t* table,
                                 int64_t table_stride, int64_t table_width, const int32_t* lengths, int64_t batch,
                                 int64_t q_heads, float* scores, popkv_stream_t stream) {
    if (const int rc = check_paged_cache(cache)) return rc;
    if (batch < 0 || batch > 65535 || q_heads <= 0 || q_heads % cache->kv_heads || table_width < 0 ||
        table_width > 0x7fffffffLL || (batch > 1 && table_stride < table_width))
        return fail(POPKV_ERR_INVALID_ARGUMENT, "invalid paged score shape");
    if (!cache->bounds) return fail(POPKV_ERR_INVALID_ARGUMENT, "paged scores need a cache with bounds");
    if (batch == 0 || table_width == 0) return POPKV_OK;
    if (!q || !table || !lengths || !scores) return fail(POPKV_ERR_INVALID_ARGUMENT, "null pointer argument");
    ScoreArgs a = {};
    a.q = q; a.bounds = cache->bounds; a.pages = cache->pages;
    a.table = table; a.table_stride = table_stride; a.width = (int)table_width; a.lengths = lengths;
    a.q_heads = (int)q_heads; a.kv_heads = (int)cache->kv_heads; a.G = (int)(q_heads / cache->kv_heads);
    a.head_dim = (int)cache->head_dim; a.page_size = (int)cache->page_size;
    a.q_vec = aligned(q, 16);
    a.scores = scores;
    // Longer walks per warp as long as they leave every SM 24 warps.
    const int64_t warps8 = (table_width + 7) / 8 * cache->kv_heads * batch;
    a.runs = 1;
    while (a.runs < 8 && warps8 / (2 * a.runs) >= 24 * (int64_t)num_sms()) a.runs *= 2;
    auto go = [&](auto kern) {
        const int per = kScoreThreads / 32 * 8 * a.runs;
        launch_pdl(kern, dim3((unsigned)((table_width + per - 1) / per), (unsigned)cache->kv_heads, (unsigned)batch),
                   dim3(kScoreThreads), 0, as_stream(stream), a);
        return check_launch("popkv_paged_score");
    };
    auto by = [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        if (cache->head_dim > 128) return go(paged_score_kernel<T, 256>);
        return cache->head_dim > 64 ? go(paged_score_kernel<T, 128>) : go(paged_score_kernel<T, 64>);
    };
    return cache->dtype == POPKV_BF16 ? by(static_cast<__nv_bfloat16*>(nullptr)) : by(static_cast<__half*>(nullptr));
}

extern "C" size_t popkv_paged_select_workspace_bytes(int64_t batch, int64_t q_heads, int64_t table_width) {
    if (batch <= 0 || q_heads <= 0 || table_width < 0) return 0;
    return (size_t)(kTicketBytes + batch * q_heads * ((table_width + 31) / 32) * 4);
}

extern "C" int popkv_paged_select(const float* scores, int64_t table_width, const int32_t* lengths, int64_t batch,
                                  int64_t q_heads, int64_t kv_heads, int64_t page_size, int64_t budget,
                                  const popkv_page_list* list, void* workspace, size_t workspace_bytes,
                                  popkv_stream_t stream) {
    if (batch < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || table_width < 0 ||
        table_width > 0x7fffffffLL / 2 || page_size <= 0 || page_size > 1024)
        return fail(POPKV_ERR_INVALID_ARGUMENT, "invalid paged select shape");
    if (budget < 1) return fail(POPKV_ERR_INVALID_ARGUMENT, "the budget must hold the newest page");
    const int64_t G = q_heads / kv_heads;
    if (G > 32) return fail(POPKV_ERR_UNSUPPORTED, "more than 32 query heads per KV head");
    if (batch * kv_heads > kMaxItems || batch * q_heads > 0x7fffffffLL)
        return fail(POPKV_ERR_UNSUPPORTED, "too many heads and sequences for one call");
    if (batch == 0) return POPKV_OK;
    if (!list || !list->counts || (list->capacity > 0 && (!list->pages || !list->heads)) || !lengths || !workspace ||
        (table_width > 0 && !scores))
        return fail(POPKV_ERR_INVALID_ARGUMENT, "null pointer argument");
    if (!aligned(workspace, 16)) return fail(POPKV_ERR_ALIGNMENT, "paged select workspace needs 16-byte alignment");
    const int64_t need = budget > table_width / G ? table_width : budget * G;
    if (list->capacity < need) return fail(POPKV_ERR_CAPACITY, "page list capacity %lld < %lld", (long long)list->capacity, (long long)need);
    if (workspace_bytes < popkv_paged_select_workspace_bytes(batch, q_heads, table_width))
        return fail(POPKV_ERR_WORKSPACE, "paged select workspace too small");
    SelectArgs a = {};
    a.scores = scores; a.width = (int)table_width; a.lengths = lengths;
    a.q_heads = (int)q_heads; a.kv_heads = (int)kv_heads; a.page_size = (int)page_size;
    a.budget = (int)imin64(budget, 0x7fffffffLL);
    a.list = *list;
    a.tickets = static_cast<uint32_t*>(workspace);
    a.bitmaps = reinterpret_cast<uint32_t*>(static_cast<char*>(workspace) + kTicketBytes);
    a.words = (int)((table_width + 31) / 32);
    auto go = [&](auto kern, int threads) {
        launch_pdl(kern, dim3((unsigned)(batch * q_heads)), dim3((unsigned)threads), 0, as_stream(stream), a);
        return check_launch("popkv_paged_select");
    };
    // Few keys per thread while the row is short (latency); 32 fill the register file.
    if (table_width <= 1024) return go(paged_select_kernel<256, 4>, 256);
    if (table_width <= 4096) return go(paged_select_kernel<512, 8>, 512);
    if (table_width <= 8192) return go(paged_select_kernel<512, 16>, 512);
    if (table_width <= 32768) return go(paged_select_kernel<1024, 32>, 1024);
    return go(paged_select_kernel<1024, 0>, 1024);
}
