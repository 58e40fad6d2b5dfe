// Writing and reading a paged key-value cache, and the per-head norm + rotary
// embedding of the rows that go into it.
//
// All of it is streaming: a row of a head is read once, normalised, rotated and
// quantised in registers by head_dim / 16 neighbouring lanes, and written once.  The floor is
// HBM (6.55 TB/s measured); what holds the kernels above it are bytes in flight and, for the
// 8-bit writers, instructions: 21 an element, of which the quotient is 3.
//
//  * norm_rope_kernel    rows of queries and keys, a warp per row and run of heads.  8192 rows of
//                        32 + 8 heads of 128 (bf16, norms and rotation): 34 us, 5.1 TB/s
//  * token_kernel        one row per sequence (a decode step): a lane group per head for
//                        queries, keys and values together, bounds widened in place; one launch's
//                        latency up to some hundred sequences: 96 rows of 32 + 2 x 8 heads of 128 in a
//                        CUDA graph 3.7 us (16-bit) and 3.9 us (8-bit), norm_rope and a write 5.9 and 6.0 us
//  * page_kernel         many rows per sequence: one CTA owns a page of some KV heads, so the
//                        page's bounds have one writer.  32768 rows of 8 heads of 128 with bounds:
//                        16-bit 50 us (5.5 TB/s), e4m3 51 us, int8 53 us (4.0 TB/s).  Fused with norm and
//                        rotation (16384 rows of 32 + 2 x 8 heads, both launches) 94 us at 16 bits and 106 us at 8,
//                        more than norm_rope and a write (90 and 94): the multipliers are made for every head
//  * read_kernel         rows back to 16 bits: the same rows from e4m3 39 us (5.2 TB/s)
#include <cmath>
#include <type_traits>

#include "paged_core.cuh"

namespace popkv {

int check_paged_cache(const popkv_paged_cache* c) {
    if (!c) return fail(POPKV_ERR_INVALID_ARGUMENT, "null cache");
    if (c->dtype != POPKV_F16 && c->dtype != POPKV_BF16)
        return fail(POPKV_ERR_UNSUPPORTED, "paged cache dtype %d is not fp16/bf16", c->dtype);
    if (c->store != POPKV_STORE_SAME && c->store != POPKV_STORE_INT8 && c->store != POPKV_STORE_E4M3)
        return fail(POPKV_ERR_UNSUPPORTED, "paged cache store %d is unknown", c->store);
    if (c->pages <= 0 || c->pages > 0x7fffffffLL || c->kv_heads <= 0 || c->kv_heads > 65535)
        return fail(POPKV_ERR_INVALID_ARGUMENT, "paged cache needs pages and kv_heads in range");
    if (c->page_size <= 0 || c->page_size % 16 || c->page_size > 1024)
        return fail(POPKV_ERR_UNSUPPORTED, "page_size %lld is not a multiple of 16 up to 1024", (long long)c->page_size);
    if (c->head_dim <= 0 || c->head_dim % 16 || c->head_dim > 256)
        return fail(POPKV_ERR_UNSUPPORTED, "paged head_dim %lld is not a multiple of 16 up to 256", (long long)c->head_dim);
    if (!c->keys || !c->values) return fail(POPKV_ERR_INVALID_ARGUMENT, "null pool pointer");
    const int64_t es = c->store == POPKV_STORE_SAME ? 2 : 1;
    if (es == 1 && (!c->key_scale || !c->value_scale))
        return fail(POPKV_ERR_INVALID_ARGUMENT, "an 8-bit paged cache needs key_scale and value_scale");
    if (c->page_stride <= 0 || c->head_stride <= 0 || c->slot_stride < c->head_dim)
        return fail(POPKV_ERR_INVALID_ARGUMENT, "paged cache strides must be positive, slots head_dim apart or more");
    if (!aligned(c->keys, 16) || !aligned(c->values, 16) || (c->page_stride * es) % 16 || (c->head_stride * es) % 16 ||
        (c->slot_stride * es) % 16 || (c->bounds && !aligned(c->bounds, 16)))
        return fail(POPKV_ERR_ALIGNMENT, "paged cache pools, bounds and strides need 16-byte alignment");
    if (es == 1 && (!aligned(c->key_scale, 16) || !aligned(c->value_scale, 16)))
        return fail(POPKV_ERR_ALIGNMENT, "paged cache scales need 16-byte alignment");
    return POPKV_OK;
}

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr uint32_t kFull = 0xffffffffu;

struct RowsIn {
    const void* data;
    int64_t row_stride, head_stride;
    bool vec;  // 16-byte loads are possible
};

struct NormRope {
    const void* q_weight;
    const void* k_weight;
    const void* cos;
    const void* sin;
    int64_t positions;
    int rotary;
    bool f32, interleaved, w_vec;
    float eps, inv_dim;
};

// What a row's elements are multiplied by, weights and table values combined (a weight of 1
// without a norm): with partner p, z_a = a aa - p ab, z_b = b bb + p ba in rotate-half form, and in the
// interleaved form z_i = x_i xx_i -+ x_partner xp_i inside each run.
struct Turn {
    float aa[8], ab[8], ba[8], bb[8];
};

template <typename T>
__device__ __forceinline__ void make_turn(Turn& t, const NormRope& n, const T* weight, const Slice& s, bool live,
                                          bool rotated, int64_t pos) {
    float wa[8], wb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) wa[i] = wb[i] = 1.0f;
    if (live && weight != nullptr) {
        load8<T>(wa, weight + s.ia, n.w_vec);
        load8<T>(wb, weight + s.ib, n.w_vec);
    }
    if (!rotated) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            t.aa[i] = wa[i];
            t.bb[i] = wb[i];
            t.ab[i] = t.ba[i] = 0.0f;
        }
        return;
    }
    float ca[8], cb[8], sa[8], sb[8];
    pos = pos < 0 ? 0 : (pos >= n.positions ? n.positions - 1 : pos);
    const int64_t at = pos * n.rotary;
    if (n.f32) {
        const float* c = static_cast<const float*>(n.cos) + at;
        const float* d = static_cast<const float*>(n.sin) + at;
        load8(ca, c + s.ia); load8(cb, c + s.ib);
        load8(sa, d + s.ia); load8(sb, d + s.ib);
    } else {
        const T* c = static_cast<const T*>(n.cos) + at;
        const T* d = static_cast<const T*>(n.sin) + at;
        load8<T>(ca, c + s.ia, true); load8<T>(cb, c + s.ib, true);
        load8<T>(sa, d + s.ia, true); load8<T>(sb, d + s.ib, true);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        t.aa[i] = wa[i] * ca[i];
        t.bb[i] = wb[i] * cb[i];
        t.ab[i] = (n.interleaved ? wa[i ^ 1] : wb[i]) * sa[i];
        t.ba[i] = (n.interleaved ? wb[i ^ 1] : wa[i]) * sb[i];
    }
}

// Norm (normed) and rotation of one row held by `group` lanes (xor shuffles below `group` stay
// inside it); lanes past head_dim / 16 hold zeros.  fp32, with every operation spelt out so that
// all kernels round alike.  Collective over the warp where n has weights.
__device__ __forceinline__ void apply_turn(Slice& s, const Turn& t, const NormRope& n, bool normed, bool rotated, int group) {
    float inv = 1.0f;
    if (n.q_weight != nullptr || n.k_weight != nullptr) {
        float ss[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            ss[0] = fmaf(s.a[i], s.a[i], ss[0]);
            ss[1] = fmaf(s.b[i], s.b[i], ss[1]);
        }
        float sum = ss[0] + ss[1];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
            if (o < group) sum += __shfl_xor_sync(kFull, sum, o);
        if (normed) inv = rsqrtf(fmaf(sum, n.inv_dim, n.eps));
    }
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a[i] = __fmul_rn(s.a[i], t.aa[i]);
        b[i] = __fmul_rn(s.b[i], t.bb[i]);
    }
    if (rotated) {
        if (n.interleaved) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                a[i] = fmaf(-s.a[i + 1], t.ab[i], a[i]);
                a[i + 1] = fmaf(s.a[i], t.ab[i + 1], a[i + 1]);
                b[i] = fmaf(-s.b[i + 1], t.ba[i], b[i]);
                b[i + 1] = fmaf(s.b[i], t.ba[i + 1], b[i + 1]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                a[i] = fmaf(-s.b[i], t.ab[i], a[i]);
                b[i] = fmaf(s.a[i], t.ba[i], b[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s.a[i] = __fmul_rn(a[i], inv);
        s.b[i] = __fmul_rn(b[i], inv);
    }
}

template <typename T>
__device__ __forceinline__ void load_slice(Slice& s, const RowsIn& in, int64_t row, int head, bool live) {
    if (live) {
        const T* p = static_cast<const T*>(in.data) + row * in.row_stride + head * in.head_stride;
        load8<T>(s.a, p + s.ia, in.vec);
        load8<T>(s.b, p + s.ib, in.vec);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) s.a[i] = s.b[i] = 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void round_slice(Slice& s) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        s.a[i] = to_float<T>(from_float<T>(s.a[i]));
        s.b[i] = to_float<T>(from_float<T>(s.b[i]));
    }
}

// Largest magnitude of a slice as an integer maximum of the bits: NaN ranks above infinity.
__device__ __forceinline__ uint32_t slice_magnitude(const Slice& s) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        top = max(top, max(__float_as_uint(s.a[i]) & 0x7fffffffu, __float_as_uint(s.b[i]) & 0x7fffffffu));
    return top;
}

// Stores one row (already rounded to T) of a head at element `at` of the pool, its scale at scales[scale_at];
// collective over the lane group.  top: the lane's largest magnitude (8-bit stores).
template <typename T, int STORE>
__device__ __forceinline__ void store_row(const Slice& s, uint32_t top, void* pool, int64_t at, float* scales,
                                          int64_t scale_at, bool live, bool leader, int group) {
    if constexpr (STORE == POPKV_STORE_SAME) {
        if (live) {
            store8<T>(static_cast<T*>(pool) + at + s.ia, s.a, true);
            store8<T>(static_cast<T*>(pool) + at + s.ib, s.b, true);
        }
    } else {
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
            if (o < group) top = max(top, __shfl_xor_sync(kFull, top, o));
        const float scale = scale_of<STORE>(__uint_as_float(top));
        if (live) {
            uint8_t* p = static_cast<uint8_t*>(pool) + at;
            const uint4 w = codes16<STORE>(s.a, s.b, scale);
            if (s.ib == s.ia + 8) {  // neighbours: 16 codes at once
                *reinterpret_cast<uint4*>(p + s.ia) = w;
            } else {
                *reinterpret_cast<uint2*>(p + s.ia) = make_uint2(w.x, w.y);
                *reinterpret_cast<uint2*>(p + s.ib) = make_uint2(w.z, w.w);
            }
            if (leader) scales[scale_at] = scale;
        }
    }
}
__device__ __forceinline__ int64_t element_of(const PagedView& c, int64_t page, int head, int slot) {
    return page * c.page_stride + head * c.head_stride + slot * c.slot_stride;
}
__device__ __forceinline__ int64_t scale_index(const PagedView& c, int64_t page, int head, int slot) {
    return (page * c.kv_heads + head) * c.page_size + slot;
}

// Largest magnitude of 16 packed 16-bit elements, as fp32 bits; NaN above infinity.
template <typename T>
__device__ __forceinline__ uint32_t top_magnitude(const uint4& x, const uint4& y) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    T2 top = *reinterpret_cast<const T2*>(&w[0]);
    top = __habs2(top);
#pragma unroll
    for (int i = 1; i < 8; ++i) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const T2*>(&w[i])));
    const uint32_t a = __float_as_uint(to_float<T>(top.x)) & 0x7fffffffu, b = __float_as_uint(to_float<T>(top.y)) & 0x7fffffffu;
    return a > b ? a : b;
}

// Minimum and maximum that keep a NaN, as amin/amax do.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T>
__device__ __forceinline__ T* bounds_of(const PagedView& c, int64_t page, int head) {
    return static_cast<T*>(c.bounds) + (page * c.kv_heads + head) * 2 * c.head_dim;
}

// First row of sequence b, kept inside the rows that exist.
__device__ __forceinline__ int64_t row_offset(const PagedRows& r, int b) {
    const int64_t o = r.offsets ? r.offsets[b] : b;
    return o < 0 ? 0 : (o > r.rows ? r.rows : o);
}

// Last sequence whose key(b) <= value, key not decreasing (0 where none is): 32 probes at a time, so a
// batch of 1024 takes two dependent loads.  Collective over the warp, value alike in all lanes.
template <typename Key>
__device__ __forceinline__ int find_sequence(int batch, int64_t value, Key&& key) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = batch;  // the answer is in [lo, hi)
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int probe = lo + lane * step;
        const uint32_t below = __ballot_sync(kFull, probe < hi && key(probe) <= value);
        if (below == 0u) return lo;
        // Keys that are not in order (no promise is made for them) still end the search.
        const int at = 31 - __clz(below);
        lo += at * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// Sequence and position of a row; position -1 where no sequence holds it.  Collective over the warp.
__device__ __forceinline__ int64_t position_of_row(const PagedRows& r, int64_t row, int& b) {
    b = r.offsets == nullptr ? static_cast<int>(row)
                             : find_sequence(r.batch, row, [&](int i) { return row_offset(r, i); });
    const int64_t first = row_offset(r, b), start = r.starts[b];
    return start >= 0 && row >= first && row < row_offset(r, b + 1) ? start + (row - first) : -1;
}

// ------------------------------------------------------------------ norm + rope
// A warp per row and run of heads, query heads first; GROUP lanes per head.  What the elements are
// multiplied by is made once for the row's queries and once for its keys.  Every lane keeps kRing steps
// of its own slices on their way through shared memory (asynchronous 16-byte copies that only it
// waits for): registers alone hold too few bytes in flight.
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
template <typename T, int GROUP>
__global__ void __launch_bounds__(kThreads, 5)
norm_rope_kernel(RowsIn q, RowsIn k, NormRope n, const int32_t* positions, PagedRows r, int64_t rows, int q_heads,
                 int kv_heads, int head_dim, int heads_per_warp, T* q_out, T* k_out, bool out_vec) {
    pdl_trigger();
    pdl_wait();
    constexpr int kStep = 32 / GROUP, kRing = 4;
    __shared__ uint4 s_ring[kRing][2][kThreads];
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int j = lane & (GROUP - 1), mine = lane / GROUP;
    const bool lives = j < head_dim / 16;
    const bool rotated = j < n.rotary / 16;
    Slice s;
    slice_runs(s, j, n.rotary, n.interleaved);
    int64_t pos = 0;
    if (positions != nullptr) {
        pos = positions[row];
    } else if (r.starts != nullptr) {  // rows of a paged cache
        int b;
        pos = position_of_row(r, row, b);
    }
    const int h0 = blockIdx.y * heads_per_warp;
    const int h1 = min(q_heads + kv_heads, h0 + heads_per_warp);
#pragma unroll 1
    for (int kind = 0; kind < 2; ++kind) {  // queries, keys
        const int lo = kind == 0 ? h0 : max(h0, q_heads) - q_heads;
        const int hi = kind == 0 ? min(h1, q_heads) : h1 - q_heads;
        if (lo >= hi) continue;
        const RowsIn& in = kind == 0 ? q : k;
        const T* weight = static_cast<const T*>(kind == 0 ? n.q_weight : n.k_weight);
        const T* src = static_cast<const T*>(in.data) + row * in.row_stride + (lo + mine) * in.head_stride;
        T* dst = (kind == 0 ? q_out + (row * q_heads + lo + mine) * head_dim : k_out + (row * kv_heads + lo + mine) * head_dim);
        const int64_t src_step = kStep * in.head_stride;
        auto fetch = [&](int h, int at) {  // heads of step h into ring entry `at`
            if (lives && h + mine < hi) {
                if (in.vec) {
                    copy16_async(smem_addr(&s_ring[at][0][threadIdx.x]), src + s.ia);
                    copy16_async(smem_addr(&s_ring[at][1][threadIdx.x]), src + s.ib);
                } else {
                    s_ring[at][0][threadIdx.x] = load_raw8<T>(src + s.ia, false);
                    s_ring[at][1][threadIdx.x] = load_raw8<T>(src + s.ib, false);
                }
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
            src += src_step;
        };
#pragma unroll
        for (int i = 0; i < kRing - 1; ++i) fetch(lo + i * kStep, i);
        Turn t;
        make_turn<T>(t, n, weight, s, lives, rotated, pos);
        int at = 0;
        for (int h = lo; h < hi; h += kStep) {
            fetch(h + (kRing - 1) * kStep, (at + kRing - 1) % kRing);
            asm volatile("cp.async.wait_group %0;\n" ::"n"(kRing - 1) : "memory");
            uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
            if (lives && h + mine < hi) {
                x = s_ring[at][0][threadIdx.x];
                y = s_ring[at][1][threadIdx.x];
            }
            at = (at + 1) % kRing;
            unpack8<T>(s.a, x);
            unpack8<T>(s.b, y);
            apply_turn(s, t, n, weight != nullptr, rotated, GROUP);
            if (lives && h + mine < hi) {
                store8<T>(dst + s.ia, s.a, out_vec);
                store8<T>(dst + s.ib, s.b, out_vec);
            }
            dst += kStep * head_dim;
        }
    }
}

// ---------------------------------------------------- one row per sequence
// Head tasks of sequence b: q_heads queries (fused calls), kv_heads keys, kv_heads values.
template <typename T, int STORE>
__global__ void __launch_bounds__(kThreads)
token_kernel(RowsIn q, RowsIn k, RowsIn v, NormRope n, PagedView c, PagedRows r, int q_heads, int group, bool fused,
             T* q_out, bool out_vec) {
    pdl_trigger();
    pdl_wait();
    const int b = blockIdx.x;
    const int lane = threadIdx.x & 31;
    const int j = lane & (group - 1);
    const int task = blockIdx.y * (kThreads / group) + static_cast<int>(threadIdx.x) / group;
    const int tasks = q_heads + 2 * c.kv_heads;
    const bool live = j < c.head_dim / 16 && task < tasks;
    const int64_t pos = r.starts[b];
    const int64_t page = page_of(r, c, b, pos);
    const bool is_q = task < q_heads;
    const bool is_k = !is_q && task < q_heads + c.kv_heads;
    const int head = is_q ? task : task - q_heads - (is_k ? 0 : c.kv_heads);
    Slice s;
    slice_runs(s, j, n.rotary, n.interleaved);
    load_slice<T>(s, is_q ? q : (is_k ? k : v), b, head, live);
    if (fused) {
        const bool turned = is_q || is_k;
        const bool rotated = turned && j < n.rotary / 16;
        const T* w = turned ? static_cast<const T*>(is_q ? n.q_weight : n.k_weight) : nullptr;
        Turn t;
        make_turn<T>(t, n, w, s, live, rotated, pos);
        apply_turn(s, t, n, w != nullptr, rotated, group);
        round_slice<T>(s);
    }
    const int slot = page >= 0 ? static_cast<int>(pos % c.page_size) : 0;
    const bool kept = live && !is_q && page >= 0;
    store_row<T, STORE>(s, slice_magnitude(s), is_k ? c.keys : c.values, element_of(c, page < 0 ? 0 : page, head, slot),
                        is_k ? c.key_scale : c.value_scale, scale_index(c, page < 0 ? 0 : page, head, slot), kept, j == 0, group);
    if (live && is_q) {
        T* o = q_out + (static_cast<int64_t>(b) * q_heads + head) * c.head_dim;
        store8<T>(o + s.ia, s.a, out_vec);
        store8<T>(o + s.ib, s.b, out_vec);
    }
    if (kept && is_k && c.bounds != nullptr) {
        T* lo = bounds_of<T>(c, page, head);
        T* hi = lo + c.head_dim;
        Slice m = s, x = s;
        if (slot != 0) {
            Slice o;
            load8<T>(o.a, lo + s.ia, true);
            load8<T>(o.b, lo + s.ib, true);
#pragma unroll
            for (int i = 0; i < 8; ++i) { m.a[i] = min_nan(m.a[i], o.a[i]); m.b[i] = min_nan(m.b[i], o.b[i]); }
            load8<T>(o.a, hi + s.ia, true);
            load8<T>(o.b, hi + s.ib, true);
#pragma unroll
            for (int i = 0; i < 8; ++i) { x.a[i] = max_nan(x.a[i], o.a[i]); x.b[i] = max_nan(x.b[i], o.b[i]); }
        }
        store8<T>(lo + s.ia, m.a, true);
        store8<T>(lo + s.ib, m.b, true);
        store8<T>(hi + s.ia, x.a, true);
        store8<T>(hi + s.ib, x.b, true);
    }
}

// --------------------------------------------------- many rows per sequence
// Work items: sequence b holds items floor(offsets[b] / P) + 2 b up to the next
// sequence's, at least floor(n / P) + 2 of them, which covers the pages that n rows from
// any start touch; the host knows their total without reading the offsets.
//
// Plain writes bring the rows of a pass through a ring of three stages in shared memory by asynchronous
// copies, one barrier a pass; the bounds are read off the same stage.  Fused ones, whose keys change on the
// way, hold the next pass in registers and put the finished keys into shared memory for the bounds.
template <typename T, int STORE, bool FUSED>
__global__ void __launch_bounds__(kThreads, FUSED ? 4 : 7)
page_kernel(RowsIn k, RowsIn v, NormRope n, PagedView c, PagedRows r, int group, int heads_per_cta) {
    pdl_trigger();
    pdl_wait();
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    extern __shared__ __align__(16) unsigned char s_raw[];
    T* s_key = reinterpret_cast<T*>(s_raw);  // [kThreads / group][head_dim], fused: the pass's keys
    const int P = c.page_size, D = c.head_dim;
    const int64_t item = blockIdx.x;
    const int b = find_sequence(r.batch, item, [&](int i) { return row_offset(r, i) / P + 2 * static_cast<int64_t>(i); });
    const int64_t r0 = row_offset(r, b), count = row_offset(r, b + 1) - r0, start = r.starts[b];
    if (start < 0) return;
    const int64_t column = start / P + item - (r0 / P + 2 * static_cast<int64_t>(b));
    const int64_t t0 = max(start, column * P), t1 = min(start + count, (column + 1) * P);
    if (t0 >= t1) return;
    const int64_t page = page_of(r, c, b, column * P);
    if (page < 0) return;
    const int lane = threadIdx.x & 31;
    const int j = lane & (group - 1);
    const bool lives = j < D / 16;
    const bool rotated = FUSED && j < n.rotary / 16;
    const int per_pass = kThreads / group;
    const int mine = static_cast<int>(threadIdx.x) / group;
    Slice s, val;
    slice_runs(s, j, FUSED ? n.rotary : 0, n.interleaved);
    val.ia = s.ia;
    val.ib = s.ib;
    const int h0 = blockIdx.y * heads_per_cta, h1 = min(c.kv_heads, h0 + heads_per_cta);
    const int d = 2 * threadIdx.x;  // thread d / 2 < D / 2 keeps the bounds of channels d and d + 1
    T2 low, high;
    auto clear_bounds = [&]() {
        low.x = low.y = from_float<T>(INFINITY);
        high.x = high.y = from_float<T>(-INFINITY);
    };
    auto widen_bounds = [&](const T* keys, int64_t t) {
        const int rows = static_cast<int>(min(static_cast<int64_t>(per_pass), t1 - t));
#pragma unroll 4
        for (int i = 0; i < rows; ++i) {
            const T2 x = *reinterpret_cast<const T2*>(keys + i * D + d);
            low = __hmin2_nan(low, x);
            high = __hmax2_nan(high, x);
        }
    };
    auto keep_bounds = [&](int head) {
        T2* lp = reinterpret_cast<T2*>(bounds_of<T>(c, page, head) + d);
        T2* hp = reinterpret_cast<T2*>(bounds_of<T>(c, page, head) + D + d);
        if (t0 != column * P) {  // the page's earlier slots were written before
            low = __hmin2_nan(low, *lp);
            high = __hmax2_nan(high, *hp);
        }
        *lp = low;
        *hp = high;
    };
    const bool bounding = c.bounds != nullptr && d < D;
    if constexpr (!FUSED) {
        constexpr int kRing = 3;
        const int tile = per_pass * D;  // elements of a pass
        const int passes = static_cast<int>((t1 - t0 + per_pass - 1) / per_pass);
        const int total = (h1 - h0) * passes;
        int next_head = h0, next_pass = 0, next_stage = 0;
        // This thread's row of the first pass, in the next head.
        const T* k_at = static_cast<const T*>(k.data) + (r0 + (t0 + mine - start)) * k.row_stride + h0 * k.head_stride + s.ia;
        const T* v_at = static_cast<const T*>(v.data) + (r0 + (t0 + mine - start)) * v.row_stride + h0 * v.head_stride + s.ia;
        auto issue = [&]() {
            if (lives && next_head < h1 && t0 + static_cast<int64_t>(next_pass) * per_pass + mine < t1) {
                const T* kp = k_at + static_cast<int64_t>(next_pass * per_pass) * k.row_stride;
                const T* vp = v_at + static_cast<int64_t>(next_pass * per_pass) * v.row_stride;
                T* to = s_key + next_stage * 2 * tile + mine * D + s.ia;
                if (k.vec && v.vec) {
                    copy16_async(smem_addr(to), kp);
                    copy16_async(smem_addr(to + 8), kp + 8);
                    copy16_async(smem_addr(to + tile), vp);
                    copy16_async(smem_addr(to + tile + 8), vp + 8);
                } else {
                    *reinterpret_cast<uint4*>(to) = load_raw8<T>(kp, k.vec);
                    *reinterpret_cast<uint4*>(to + 8) = load_raw8<T>(kp + 8, k.vec);
                    *reinterpret_cast<uint4*>(to + tile) = load_raw8<T>(vp, v.vec);
                    *reinterpret_cast<uint4*>(to + tile + 8) = load_raw8<T>(vp + 8, v.vec);
                }
            }
            asm volatile("cp.async.commit_group;\n" ::: "memory");
            if (++next_pass == passes) {
                next_pass = 0;
                ++next_head;
                k_at += k.head_stride;
                v_at += v.head_stride;
            }
            next_stage = next_stage + 1 == kRing ? 0 : next_stage + 1;
        };
        issue();
        issue();
        int head = h0, pass = 0, stage = 0;
        int64_t at = element_of(c, page, h0, 0);         // of the head's slot 0
        int64_t scale_at = scale_index(c, page, h0, 0);
        clear_bounds();
        for (int it = 0; it < total; ++it) {
            asm volatile("cp.async.wait_group 1;\n" ::: "memory");
            __syncthreads();  // this stage has landed for every thread, and the stage before it has been read
            issue();
            const int64_t t = t0 + static_cast<int64_t>(pass) * per_pass;
            const bool live = lives && t + mine < t1;
            const int slot = static_cast<int>(t + mine - column * P);
            const T* keys = s_key + stage * 2 * tile;
            uint4 x = make_uint4(0u, 0u, 0u, 0u), y = x;
            if (live) {
                x = *reinterpret_cast<const uint4*>(keys + mine * D + s.ia);
                y = *reinterpret_cast<const uint4*>(keys + mine * D + s.ib);
            }
            unpack8<T>(s.a, x);
            unpack8<T>(s.b, y);
            const int64_t to = at + slot * c.slot_stride;
            store_row<T, STORE>(s, STORE == POPKV_STORE_SAME ? 0u : top_magnitude<T>(x, y), c.keys, to, c.key_scale, scale_at + slot,
                                live, j == 0, group);
            if (live) {
                x = *reinterpret_cast<const uint4*>(keys + tile + mine * D + s.ia);
                y = *reinterpret_cast<const uint4*>(keys + tile + mine * D + s.ib);
            }
            unpack8<T>(s.a, x);
            unpack8<T>(s.b, y);
            store_row<T, STORE>(s, STORE == POPKV_STORE_SAME ? 0u : top_magnitude<T>(x, y), c.values, to, c.value_scale,
                                scale_at + slot, live, j == 0, group);
            if (bounding) widen_bounds(keys, t);
            if (++pass == passes) {
                if (bounding) keep_bounds(head);
                clear_bounds();
                pass = 0;
                ++head;
                at += c.head_stride;
                scale_at += P;
            }
            stage = stage + 1 == kRing ? 0 : stage + 1;
        }
        return;
    }
    // Passes of per_pass rows, head by head; the next pass's rows are loaded before this one's are worked on.
    uint4 kx, ky, vx, vy;
    auto fetch = [&](int64_t t, int head) {
        kx = ky = vx = vy = make_uint4(0u, 0u, 0u, 0u);
        if (!lives || head >= h1 || t + mine >= t1) return;
        const int64_t row = r0 + (t + mine - start);
        const T* p = static_cast<const T*>(k.data) + row * k.row_stride + head * k.head_stride;
        kx = load_raw8<T>(p + s.ia, k.vec);
        ky = load_raw8<T>(p + s.ib, k.vec);
        p = static_cast<const T*>(v.data) + row * v.row_stride + head * v.head_stride;
        vx = load_raw8<T>(p + s.ia, v.vec);
        vy = load_raw8<T>(p + s.ib, v.vec);
    };
    fetch(t0, h0);
    for (int head = h0; head < h1; ++head) {
        clear_bounds();
        for (int64_t t = t0; t < t1; t += per_pass) {
            const bool live = lives && t + mine < t1;
            const int slot = static_cast<int>(t + mine - column * P);
            unpack8<T>(s.a, kx);
            unpack8<T>(s.b, ky);
            uint4 key_a = kx, key_b = ky;
            const uint4 val_a = vx, val_b = vy;
            const bool last_pass = t + per_pass >= t1;
            fetch(last_pass ? t0 : t + per_pass, last_pass ? head + 1 : head);
            {
                Turn turn;
                make_turn<T>(turn, n, static_cast<const T*>(n.k_weight), s, live, rotated && live, t + mine);
                apply_turn(s, turn, n, n.k_weight != nullptr, rotated && live, group);
                key_a = pack8<T>(s.a);
                key_b = pack8<T>(s.b);
                unpack8<T>(s.a, key_a);  // as they were rounded
                unpack8<T>(s.b, key_b);
            }
            store_row<T, STORE>(s, STORE == POPKV_STORE_SAME ? 0u : top_magnitude<T>(key_a, key_b), c.keys,
                                element_of(c, page, head, slot), c.key_scale, scale_index(c, page, head, slot), live, j == 0, group);
            if (c.bounds != nullptr && live) {
                *reinterpret_cast<uint4*>(s_key + mine * D + s.ia) = key_a;
                *reinterpret_cast<uint4*>(s_key + mine * D + s.ib) = key_b;
            }
            unpack8<T>(val.a, val_a);
            unpack8<T>(val.b, val_b);
            store_row<T, STORE>(val, STORE == POPKV_STORE_SAME ? 0u : top_magnitude<T>(val_a, val_b), c.values,
                                element_of(c, page, head, slot), c.value_scale, scale_index(c, page, head, slot), live, j == 0, group);
            if (c.bounds != nullptr) {
                __syncthreads();
                if (bounding) widen_bounds(s_key, t);
                __syncthreads();
            }
        }
        if (bounding) keep_bounds(head);
    }
}

// ------------------------------------------------------------------------ read
template <typename T, int STORE>
__global__ void __launch_bounds__(kThreads)
read_kernel(PagedView c, PagedRows r, int group, int heads_per_warp, T* k_out, T* v_out, bool out_vec) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    if (row >= r.rows) return;
    int b;
    const int64_t pos = position_of_row(r, row, b);
    const int64_t page = page_of(r, c, b, pos);
    const int slot = page >= 0 ? static_cast<int>(pos % c.page_size) : 0;
    const int j = lane & (group - 1);
    if (j >= c.head_dim / 16) return;
    const int h0 = blockIdx.y * heads_per_warp;
    const int h1 = min(2 * c.kv_heads, h0 + heads_per_warp);  // keys, then values
    const int step = 32 / group;
    constexpr int kAhead = 4;  // loads in flight per lane
    for (int hb = h0 + lane / group; hb < h1; hb += kAhead * step) {
        Cached16<STORE> raw[kAhead];
        float scale[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int h = hb + i * step;
            scale[i] = 1.0f;
            if (h >= h1 || page < 0) continue;
            const bool is_k = h < c.kv_heads;
            const int head = is_k ? h : h - c.kv_heads;
            raw[i] = load_cached16<T, STORE>(is_k ? c.keys : c.values,
                                             page * c.page_stride + head * c.head_stride + slot * c.slot_stride + 16 * j);
            if (STORE != POPKV_STORE_SAME)
                scale[i] = (is_k ? c.key_scale : c.value_scale)[(page * c.kv_heads + head) * c.page_size + slot];
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int h = hb + i * step;
            if (h >= h1) continue;
            const bool is_k = h < c.kv_heads;
            float x[8] = {}, y[8] = {};
            if (page >= 0) unpack_cached16<T, STORE>(x, y, raw[i]);
            if (STORE != POPKV_STORE_SAME) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] *= scale[i];
                    y[e] *= scale[i];
                }
            }
            T* o = (is_k ? k_out : v_out) + (row * c.kv_heads + (is_k ? h : h - c.kv_heads)) * c.head_dim + 16 * j;
            store8<T>(o, x, out_vec);
            store8<T>(o + 8, y, out_vec);
        }
    }
}

// --------------------------------------------------------------------- host side
int lane_group(int64_t head_dim) {
    int g = 1;
    while (g * 16 < head_dim) g *= 2;
    return g;
}

RowsIn rows_in(const popkv_rows& r) {
    return RowsIn{r.data, r.row_stride, r.head_stride, aligned(r.data, 16) && r.row_stride % 8 == 0 && r.head_stride % 8 == 0};
}

int check_norm_rope(const popkv_norm_rope_args* a, int64_t head_dim, NormRope* n) {
    if (!a) return fail(POPKV_ERR_INVALID_ARGUMENT, "null norm/rope arguments");
    if (head_dim <= 0 || head_dim % 16 || head_dim > 256)
        return fail(POPKV_ERR_UNSUPPORTED, "norm_rope head_dim %lld is not a multiple of 16 up to 256", (long long)head_dim);
    if (a->rotary_dim < 0 || a->rotary_dim % 16 || a->rotary_dim > head_dim)
        return fail(POPKV_ERR_UNSUPPORTED, "rotary_dim %lld is not a multiple of 16 up to head_dim", (long long)a->rotary_dim);
    if (a->rotary_dim > 0 && (!a->cos || !a->sin || a->positions <= 0))
        return fail(POPKV_ERR_INVALID_ARGUMENT, "a rotation needs cos and sin tables");
    if (a->rotary_dim > 0 && (!aligned(a->cos, 16) || !aligned(a->sin, 16)))
        return fail(POPKV_ERR_ALIGNMENT, "cos and sin tables need 16-byte alignment");
    if (!(a->eps >= 0.0f)) return fail(POPKV_ERR_INVALID_ARGUMENT, "eps must not be negative");
    n->q_weight = a->q_weight;
    n->k_weight = a->k_weight;
    n->cos = a->cos;
    n->sin = a->sin;
    n->positions = a->positions;
    n->rotary = (int)a->rotary_dim;
    n->f32 = a->tables_f32 != 0;
    n->interleaved = a->interleaved != 0;
    n->w_vec = aligned(a->q_weight, 16) && aligned(a->k_weight, 16);  // NULL counts as aligned
    n->eps = a->eps;
    n->inv_dim = 1.0f / (float)head_dim;
    return POPKV_OK;
}

int check_rows(const popkv_paged_cache* cache, const int32_t* table, int64_t table_stride, int64_t table_width,
               const int32_t* starts, const int32_t* row_offsets, int64_t batch, int64_t rows, PagedRows* r) {
    if (batch < 0 || rows < 0 || batch > 0x3fffffffLL || rows > 0x7fffffffLL || table_width < 0 ||
        table_width > 0x7fffffffLL || (batch > 1 && table_stride < table_width))
        return fail(POPKV_ERR_INVALID_ARGUMENT, "invalid batch, rows or block table size");
    if (!row_offsets && rows != batch)
        return fail(POPKV_ERR_INVALID_ARGUMENT, "without row_offsets there is one row per sequence");
    if (rows > 0 && batch == 0) return fail(POPKV_ERR_INVALID_ARGUMENT, "rows without sequences");
    if (batch > 0 && rows > 0 && (!starts || (table_width > 0 && !table)))
        return fail(POPKV_ERR_INVALID_ARGUMENT, "null block table or starts");
    r->table = table;
    r->table_stride = table_stride;
    r->table_width = (int)table_width;
    r->starts = starts;
    r->offsets = row_offsets;
    r->batch = (int)batch;
    r->rows = rows;
    (void)cache;
    return POPKV_OK;
}

template <typename F>
int by_store(int dtype, int store, F&& f) {
    auto go = [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        switch (store) {
            case POPKV_STORE_INT8: return f(tp, std::integral_constant<int, POPKV_STORE_INT8>{});
            case POPKV_STORE_E4M3: return f(tp, std::integral_constant<int, POPKV_STORE_E4M3>{});
            default: return f(static_cast<T*>(nullptr), std::integral_constant<int, POPKV_STORE_SAME>{});
        }
    };
    return dtype == POPKV_BF16 ? go(static_cast<__nv_bfloat16*>(nullptr)) : go(static_cast<__half*>(nullptr));
}

// Heads that one warp walks: enough warps to fill the GPU first, then as many heads as
// share the row's tables.
int heads_per_warp(int64_t rows, int heads, int group) {
    const int step = 32 / group;
    int hpw = (heads + step - 1) / step * step;
    const int64_t wanted = (int64_t)num_sms() * 32;
    while (hpw > step && rows * ((heads + hpw - 1) / hpw) < wanted) hpw = (hpw / 2 + step - 1) / step * step;
    return hpw;
}

int launch_norm_rope(const popkv_rows& q, const popkv_rows& k, const NormRope& n, const int32_t* positions,
                     const PagedRows& r, int dtype, int64_t rows, int q_heads, int kv_heads, int head_dim, void* q_out, void* k_out, cudaStream_t st) {
    const int group = lane_group(head_dim);
    const int hpw = heads_per_warp(rows, q_heads + kv_heads, group);
    const dim3 grid((unsigned)((rows + kWarps - 1) / kWarps), (unsigned)((q_heads + kv_heads + hpw - 1) / hpw));
    const bool out_vec = aligned(q_out, 16) && aligned(k_out, 16);
    auto go = [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        auto with = [&](auto kern) {
            launch_pdl(kern, grid, dim3(kThreads), 0, st, rows_in(q), rows_in(k), n, positions, r, rows, q_heads, kv_heads,
                       head_dim, hpw, static_cast<T*>(q_out), static_cast<T*>(k_out), out_vec);
            return check_launch("popkv_norm_rope");
        };
        switch (group) {
            case 1: return with(norm_rope_kernel<T, 1>);
            case 2: return with(norm_rope_kernel<T, 2>);
            case 4: return with(norm_rope_kernel<T, 4>);
            case 8: return with(norm_rope_kernel<T, 8>);
            default: return with(norm_rope_kernel<T, 16>);
        }
    };
    return dtype == POPKV_BF16 ? go(static_cast<__nv_bfloat16*>(nullptr)) : go(static_cast<__half*>(nullptr));
}

int launch_write(const popkv_rows& q, const popkv_rows& k, const popkv_rows& v, const NormRope& n,
                 const popkv_paged_cache* cache, const PagedRows& r, int q_heads, bool fused, void* q_out,
                 cudaStream_t st) {
    const PagedView view = paged_view(cache);
    const int group = lane_group(cache->head_dim);
    return by_store(cache->dtype, cache->store, [&](auto* tp, auto store) {
        using T = std::remove_pointer_t<decltype(tp)>;
        constexpr int S = decltype(store)::value;
        if (r.offsets == nullptr) {
            const int tasks = q_heads + 2 * view.kv_heads;
            const int per_cta = kThreads / group;
            launch_pdl(token_kernel<T, S>, dim3((unsigned)r.batch, (unsigned)((tasks + per_cta - 1) / per_cta)),
                       dim3(kThreads), 0, st, rows_in(q), rows_in(k), rows_in(v), n, view, r, q_heads, group, fused,
                       static_cast<T*>(q_out), aligned(q_out, 16));
            return check_launch("popkv_paged_write");
        }
        if (fused) {
            const int rc = launch_norm_rope(q, popkv_rows{nullptr, 0, 0}, n, nullptr, r, cache->dtype, r.rows, q_heads, 0,
                                            view.head_dim, q_out, nullptr, st);
            if (rc != POPKV_OK) return rc;
        }
        const int64_t items = r.rows / view.page_size + 2 * (int64_t)r.batch;
        if (items > 0x7fffffffLL) return fail(POPKV_ERR_UNSUPPORTED, "too many pages for one launch");
        const size_t smem = (size_t)(fused ? 1 : 6) * (kThreads / group) * view.head_dim * 2;
        // Several heads per CTA once the pages alone fill the GPU: fewer look-ups, loads run ahead.
        int hpc = 1;
        while (hpc < 4 && hpc < view.kv_heads && items * ((view.kv_heads + 2 * hpc - 1) / (2 * hpc)) >= 16 * (int64_t)num_sms()) hpc *= 2;
        launch_pdl(fused ? page_kernel<T, S, true> : page_kernel<T, S, false>,
                   dim3((unsigned)items, (unsigned)((view.kv_heads + hpc - 1) / hpc)), dim3(kThreads), smem, st, rows_in(k),
                   rows_in(v), n, view, r, group, hpc);
        return check_launch("popkv_paged_write");
    });
}

}  // namespace
}  // namespace popkv

using namespace popkv;

extern "C" int popkv_norm_rope(popkv_rows q, popkv_rows k, const popkv_norm_rope_args* args,
                               const int32_t* positions_of_rows, int dtype, int64_t rows, int64_t q_heads,
                               int64_t kv_heads, int64_t head_dim, void* q_out, void* k_out, popkv_stream_t stream) {
    NormRope n;
    if (const int rc = check_norm_rope(args, head_dim, &n)) return rc;
    if (dtype != POPKV_F16 && dtype != POPKV_BF16)
        return fail(POPKV_ERR_UNSUPPORTED, "norm_rope dtype %d is not fp16/bf16", dtype);
    if (rows < 0 || rows > 0x7fffffffLL || q_heads < 0 || kv_heads < 0 || q_heads > 65535 || kv_heads > 65535)
        return fail(POPKV_ERR_INVALID_ARGUMENT, "invalid norm_rope shape");
    if (rows == 0 || q_heads + kv_heads == 0) return POPKV_OK;
    if ((q_heads > 0 && (!q.data || !q_out)) || (kv_heads > 0 && (!k.data || !k_out)) ||
        (n.rotary > 0 && !positions_of_rows))
        return fail(POPKV_ERR_INVALID_ARGUMENT, "null pointer argument");
    return launch_norm_rope(q, k, n, positions_of_rows, PagedRows{}, dtype, rows, (int)q_heads, (int)kv_heads, (int)head_dim, q_out,
                            k_out, as_stream(stream));
}

extern "C" int popkv_paged_write(const popkv_paged_cache* cache, popkv_rows k, popkv_rows v, const int32_t* table,
                                 int64_t table_stride, int64_t table_width, const int32_t* starts,
                                 const int32_t* row_offsets, int64_t batch, int64_t rows, popkv_stream_t stream) {
    PagedRows r;
    if (const int rc = check_paged_cache(cache)) return rc;
    if (const int rc = check_rows(cache, table, table_stride, table_width, starts, row_offsets, batch, rows, &r)) return rc;
    if (rows == 0) return POPKV_OK;
    if (!k.data || !v.data) return fail(POPKV_ERR_INVALID_ARGUMENT, "null pointer argument");
    const NormRope none = {};
    return launch_write(popkv_rows{nullptr, 0, 0}, k, v, none, cache, r, 0, false, nullptr, as_stream(stream));
}

extern "C" int popkv_norm_rope_write(popkv_rows q, popkv_rows k, popkv_rows v, const popkv_norm_rope_args* args,
                                     const popkv_paged_cache* cache, const int32_t* table, int64_t table_stride,
                                     int64_t table_width, const int32_t* starts, const int32_t* row_offsets,
                                     int64_t batch, int64_t rows, int64_t q_heads, void* q_out,
                                     popkv_stream_t stream) {
    PagedRows r;
    NormRope n;
    if (const int rc = check_paged_cache(cache)) return rc;
    if (const int rc = check_norm_rope(args, cache->head_dim, &n)) return rc;
    if (const int rc = check_rows(cache, table, table_stride, table_width, starts, row_offsets, batch, rows, &r)) return rc;
    if (q_heads <= 0 || q_heads > 65535) return fail(POPKV_ERR_INVALID_ARGUMENT, "invalid q_heads");
    if (rows == 0) return POPKV_OK;
    if (!q.data || !k.data || !v.data || !q_out) return fail(POPKV_ERR_INVALID_ARGUMENT, "null pointer argument");
    return launch_write(q, k, v, n, cache, r, (int)q_heads, true, q_out, as_stream(stream));
}

extern "C" int popkv_paged_read(const popkv_paged_cache* cache, const int32_t* table, int64_t table_stride,
                                int64_t table_width, const int32_t* starts, const int32_t* row_offsets, int64_t batch,
                                int64_t rows, void* k_out, void* v_out, popkv_stream_t stream) {
    PagedRows r;
    if (const int rc = check_paged_cache(cache)) return rc;
    if (const int rc = check_rows(cache, table, table_stride, table_width, starts, row_offsets, batch, rows, &r)) return rc;
    if (rows == 0) return POPKV_OK;
    if (!k_out || !v_out) return fail(POPKV_ERR_INVALID_ARGUMENT, "null pointer argument");
    const PagedView view = paged_view(cache);
    const int group = lane_group(cache->head_dim);
    const int hpw = heads_per_warp(rows, 2 * view.kv_heads, group);
    const dim3 grid((unsigned)((rows + kWarps - 1) / kWarps), (unsigned)((2 * view.kv_heads + hpw - 1) / hpw));
    const bool out_vec = aligned(k_out, 16) && aligned(v_out, 16);
    return by_store(cache->dtype, cache->store, [&](auto* tp, auto store) {
        using T = std::remove_pointer_t<decltype(tp)>;
        launch_pdl(read_kernel<T, decltype(store)::value>, grid, dim3(kThreads), 0, as_stream(stream), view, r, group,
                   hpw, static_cast<T*>(k_out), static_cast<T*>(v_out), out_vec);
        return check_launch("popkv_paged_read");
    });
}
