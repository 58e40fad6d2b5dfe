// Decode attention of one new token per sequence over a paged cache.
//
//   s_j = scale * q . k_j,  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  lse = m + ln(sum)
//
// over the sequence's tokens (or its listed pages'), split over the length and joined in
// the same launch.  What bounds it is HBM: every cached byte is read once and used by the
// G query heads of its KV head, 2 G multiply-adds a byte at 16 bits.  Measured, 16 sequences of
// 32768 tokens, 8 KV heads of 128: 16 bits (64 query heads) 2.15 GB in 324 us (6.6 TB/s, a copy's
// rate); e4m3 (32 query heads) 1.11 GB in 184 us (6.0 TB/s); int8 in 217 us (5.1 TB/s: it takes 553 instructions
// per 16 tokens, 176 of them to turn codes into fp16 and most of the others per unit, where bf16 takes 280, and the
// issue slots bound it).  One sequence of 4096 tokens: 10.7 us, a chain of latencies (launch, lengths, table, loads,
// ticket, merge), not of bytes.
//
// Units and schedule.  The work is cut into units of 16 tokens of one page.  CTA c of a
// grid that fills the GPU once takes units [c q, (c + 1) q) of all sequences and heads laid end to
// end, with q found from the device's lengths (Schedule), so ragged batches stay balanced
// and nothing is known on the host.  A stretch of one (sequence, KV head, group of query heads)
// in a CTA is a piece; an item that one CTA covers is written directly, the others leave fp32
// partials and the CTA that takes the item's last ticket merges them in piece order (the
// same sum every time).
//
// Pipeline.  Each of the 4 warps owns a ring of unit buffers filled by TMA boxes of
// [16 rows x 128 bytes] (128-byte swizzle) on its own mbarriers: no block barrier inside a
// piece, loads run ahead across pieces.  Page numbers of the next 32 units are read by 32 lanes
// at once.
//
// Tensor cores.  mma.m16n8k16 with tokens, then channels, in M and query heads in N = 8: S^T = K Q^T,
// O^T += V^T P^T, so that nothing of a multiply is idle with 8 heads and K and V rows become A
// fragments as they lie in shared memory (16 bits: ldmatrix; 8 bits: 16-byte loads, whose channel
// order the queries follow).  P^T turns from accumulators into B fragments by movmatrix and
// enters as two 16-bit halves, a weight and its rounding residue (what that loses: Shape::kUp).
// 9 to 16 heads take the same K and V fragments twice; more heads (more than 8 above 128 channels) are items of
// their own that read the cache again: 16 x 65536 tokens, one KV head of 128, bf16: 8 heads 90 us, 16 heads 95,
// 32 heads 127, 64 heads 322; int8 73, 103, 179 us for 8, 16, 32.
//
// 8-bit caches.  Codes become exact fp16 numbers (integers by the 1024 + u pattern, e4m3
// by conversion) on their way into the fragments; queries enter as fp16 scaled by a power of
// two per head (exact but for elements far below the head's largest: load_queries); key scales multiply
// the logits in fp32.  Value scales go into the weights:
// w_j = 2^(s_j + log2 scale_j - n) with a reference n of their own, so that fp16 weights keep their
// precision whatever the scales are; the softmax sum keeps its own reference m.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>
#include <cmath>
#include <type_traits>

#include "paged_core.cuh"

namespace popkv {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr uint32_t kFull = 0xffffffffu;
constexpr int kUnit = 16;                  // tokens per unit
constexpr int kMaxItems = 65536 - 1;       // (sequence, KV head, head group) triples per call
constexpr int64_t kTicketBytes = POPKV_PAGED_TICKET_BYTES;  // tickets; the last word counts waits that ran out
static_assert(kTicketBytes == 4 * (kMaxItems + 1), "a ticket per item and the count");
constexpr int kMaxHeads = 16;              // query heads per item
constexpr int kMinUnits = 8;               // units per CTA below which a further split costs more than it gives
constexpr unsigned long long kWaitNs = 2000000000ull;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;

struct AttnArgs {
    const void* q;
    void* out;
    float* lse;
    const float* key_scale;
    const float* value_scale;
    int64_t pages;
    const int32_t* table;
    int64_t table_stride;
    int table_width;
    const int32_t* lengths;
    int batch, q_heads, kv_heads, G, head_groups, heads_per_item, head_dim, page_size;
    float sl2;   // scale * log2(e)
    bool q_vec;    // q is 16-byte aligned
    bool out_vec;  // out is 8-byte aligned
    const int32_t* list_counts;  // NULL: every page of the sequence
    const int32_t* list_pages;   // these two may be NULL where list_capacity is 0
    const uint32_t* list_heads;
    int64_t list_capacity;
    uint32_t* tickets;
    float* parts;  // [2 * grid][part_floats]
    int part_floats;
    int lost_cta;                // tests: this CTA's copies never complete (-1: none)
    unsigned long long wait_ns;  // limit of a wait for a copy
};

// ---------------------------------------------------------------- small pieces
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ float lds32f(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
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
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float lg2(float x) {
    float r;
    asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(kFull, x, 1));
    return fmaxf(x, __shfl_xor_sync(kFull, x, 2));
}
// Over the 8 lanes that hold a fragment column.
__device__ __forceinline__ float column_max(float x) {
    x = fmaxf(x, __shfl_xor_sync(kFull, x, 4));
    x = fmaxf(x, __shfl_xor_sync(kFull, x, 8));
    return fmaxf(x, __shfl_xor_sync(kFull, x, 16));
}
__device__ __forceinline__ float column_sum(float x) {
    x += __shfl_xor_sync(kFull, x, 4);
    x += __shfl_xor_sync(kFull, x, 8);
    return x + __shfl_xor_sync(kFull, x, 16);
}
// Transpose of an 8x8 matrix of 16-bit elements held as accumulator pairs.
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// Two fp32 numbers as a packed 16-bit pair, and what the rounding left.
template <bool BF16>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
    if constexpr (BF16) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
        const float rx = x - __uint_as_float(hi << 16), ry = y - __uint_as_float(hi & 0xffff0000u);
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(ry), "f"(rx));
    } else {
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        const float rx = x - h.x, ry = y - h.y;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(ry), "f"(rx));
    }
}
// ------------------------------------------------------------------- schedule
// Segments are sequences (all pages) or (sequence, KV head) lists; a segment stands for
// `reps` items of equal length.  Either the items are cut into chunks of q units, q the least that gives
// every chunk a CTA of its own; or all items are laid end to end with `gap` empty units before
// each (the price of ending a piece: two barriers, a merge, a ticket) and dealt out evenly, so that a CTA
// may hold the end of one item and the start of the next.  Chunks are taken where they leave the
// longest share hardly longer.
struct Schedule {
    int q;     // units per CTA
    int gap;   // empty units before an item; 0: chunks (item starts are multiples of q)
};
constexpr int kGap = 32;

__device__ __forceinline__ int64_t seq_length(const AttnArgs& a, int b) {
    const int64_t len = a.lengths[b], most = static_cast<int64_t>(a.table_width) * a.page_size;
    return len < 0 ? 0 : (len < most ? len : most);
}
// Units of a segment.
__device__ __forceinline__ int segment_units(const AttnArgs& a, int seg) {
    if (a.list_counts == nullptr) return static_cast<int>((seq_length(a, seg) + kUnit - 1) / kUnit);
    const int n = a.list_counts[seg];
    return (n < 0 ? 0 : (n < a.list_capacity ? n : static_cast<int>(a.list_capacity))) * (a.page_size / kUnit);
}
// Room of an item in the line of all items.
__device__ __forceinline__ int room(int units, const Schedule& s) {
    if (units == 0) return 0;
    return s.gap ? units + s.gap : (units + s.q - 1) / s.q * s.q;
}

// units: of segment `lane`, where there are at most 32 (-1: read them here).
__device__ __forceinline__ Schedule plan(const AttnArgs& a, int segs, int reps, int units, int lane, int grid) {
    int64_t sum;
    int top = 0, busy = 0;  // longest segment, segments with units
    if (segs <= 32) {
        // Fewer than 2^27 units each: the sum of 32 fits 32 bits.
        sum = __reduce_add_sync(kFull, static_cast<unsigned>(units));
        top = __reduce_max_sync(kFull, units);
        busy = __popc(__ballot_sync(kFull, units > 0));
    } else {
        sum = 0;
        for (int i = lane; i < segs; i += 32) {
            const int u = segment_units(a, i);
            sum += u;
            top = u > top ? u : top;
            busy += u > 0;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
        top = __reduce_max_sync(kFull, top);
        busy = __reduce_add_sync(kFull, busy);
    }
    sum *= reps;
    const int64_t items = static_cast<int64_t>(busy) * reps;
    const int64_t line = sum + items * kGap;
    const bool small = line + grid <= 0x7fffffff;  // 32-bit divisions
    const int64_t fair = small ? static_cast<int64_t>((static_cast<unsigned>(line) + grid - 1) / static_cast<unsigned>(grid))
                               : (line + grid - 1) / grid;
    Schedule s;
    s.gap = kGap;
    int64_t q = fair;
    if (items > 0 && 2 * items <= grid) {
        // Every item in at most grid / items chunks, or a fair share plus one chunk each.
        const unsigned n = static_cast<unsigned>(items), each = static_cast<unsigned>(grid) / n, rest = grid - n;
        const int64_t q1 = (static_cast<unsigned>(top) + each - 1) / each;
        const int64_t q2 = small ? static_cast<int64_t>((static_cast<unsigned>(sum) + rest - 1) / rest) : (sum + rest - 1) / rest;
        const int64_t c = q1 < q2 ? q1 : q2;
        if (c <= fair + fair / 32) {
            s.gap = 0;
            q = c;
        }
    }
    s.q = static_cast<int>(q < kMinUnits ? kMinUnits : q);
    return s;
}

// Bits of the heads that an item has (the last head group of a KV head may be short).
__device__ __forceinline__ uint32_t item_heads(const AttnArgs& a, int item) {
    const int left = a.G - (item % a.head_groups) * a.heads_per_item;
    return left >= a.heads_per_item ? (1u << a.heads_per_item) - 1u : (1u << left) - 1u;
}

template <typename T, int STORE, int DP, int NG>
struct Shape {
    static constexpr int kCached = STORE == POPKV_STORE_SAME ? 2 : 1;       // bytes per cached element
    static constexpr int kRowBytes = DP * kCached;
    static constexpr int kBoxBytes = kRowBytes < 128 ? kRowBytes : 128;     // per row
    static constexpr int kBoxes = kRowBytes / kBoxBytes;
    static constexpr int kBoxChannels = kBoxBytes / kCached;
    static constexpr int kPoolBytes = kUnit * kRowBytes;                    // keys (or values) of a unit
    static constexpr int kBufBytes = 2 * kPoolBytes;
    static constexpr int kScaleBytes = kCached == 1 ? 2 * kUnit * 4 : 0;
    static constexpr bool kBf16 = STORE == POPKV_STORE_SAME && std::is_same<T, __nv_bfloat16>::value;
    // Softmax weights are relative to a reference that a maximum may pass by 2^kSlack, and are held times 2^kUp as
    // two 16-bit halves.  bf16: up to 2^-16 of a weight is lost whatever its size, and with 2^-8 no weight is
    // above 1, so that sums of huge values hold.  fp16: 2^-22 of a weight or, as fp16's steps end at 2^-24,
    // 2^(-25 - kUp) of the largest.  Over 16-bit caches kUp uses fp16's whole range, 2^15 with the slack: weights
    // that a token of little value keeps far below it are the answer then.  The price is a reference that moves more
    // often: 64 sequences of 1024 tokens 33.4 us instead of 32.9, 16 of 32768 tokens no difference.  Over 8-bit
    // caches a weight has its value's scale in it, so that what is lost is little beside the largest term itself.
    static constexpr bool kHalfCache = kCached == 2 && !kBf16;
    static constexpr float kSlack = kHalfCache ? 2.0f : 8.0f;
    static constexpr float kUp = kBf16 ? -8.0f : (kHalfCache ? 13.0f : 6.0f);
    static constexpr int kTiles = DP / 16;                                  // m16 channel tiles of O^T
    static constexpr int kSteps = DP / 16;                                  // k16 channel steps of S^T
    static constexpr int kHeads = 8 * NG;
    // CTAs per SM as the accumulators' registers allow, and unit buffers per warp: 96 to 128 KB
    // of loads in flight or landed per SM, which leaves the next launch's CTAs room to start early.
    // Deeper rings were slower: with 192 KB per SM the ragged case of 16 x 32768 tokens took 169 us
    // instead of 161, 8 x 131072 over pages 152 instead of 139.
    static constexpr int kCtas = kBufBytes >= 16384 ? 1 : (kCached == 1 && NG == 1 && DP <= 128 ? (DP == 64 ? 4 : 3) : 2);
    static constexpr int kStages = kBufBytes >= 8192 ? 2
                                   : kCtas >= 3      ? (DP == 128 ? 2 : 3)
                                                     : (DP == 128 ? 3 : 4);
    static constexpr int kRing = kWarps * kStages * kBufBytes;
    static constexpr int kScales = kWarps * kStages * kScaleBytes;
    static constexpr int kMl = kWarps * kHeads * 2 * 4;
    static constexpr int kSmem = 1024 + kRing + kScales + kMl + kWarps * (kStages * (16 + 8) + 32 + 4) + 16;
    static_assert(kBufBytes >= 8 * DP * 4, "a unit buffer holds a warp's sums of 8 heads");
    static_assert((kSmem + 1024) * kCtas <= 228 * 1024 && kCtas <= 4, "shared memory per SM, workspace");
};

// What a warp's ring entry holds: a unit (tokens > 0) or the end of a piece.
struct alignas(16) Entry {
    int tokens;      // 1..16; 0: end of the piece; -1: end of the CTA's last piece
    uint32_t heads;  // unit: heads of the item that attend it.  End: first CTA of the item
    int item;
    int last;        // end: last CTA of the item
};

// Walks the pieces of this CTA and the units of one warp in them; alike in all lanes but
// for the look-ahead, in which lane i holds the warp's i-th next unit.
struct Producer {
    int base, end;     // first unit of the look-ahead, end of the piece
    uint32_t live;     // lanes whose unit is mapped and not yet loaded
    int item, kvh, b;
    int64_t len;       // tokens of the sequence
    int page, info;    // per lane: page, slot | tokens << 16
    int next_page;     // per lane: table entry of the following look-ahead (whole sequences), read early
    uint32_t heads;
    bool done, fresh;  // no piece left; the piece has not been looked at yet
};
// What only the ends of pieces need, one per warp in shared memory.
struct Walk {
    int64_t virt;      // room before the current item (its gap included)
    int seg, rep;
    int item_units;
    int u0;            // the piece's first unit
    int left;          // room of the CTA's share behind the piece's start
    int turn;          // which warp takes the piece's first unit
};

template <typename T, int STORE, int DP, int NG>
__global__ void __launch_bounds__(kThreads, (Shape<T, STORE, DP, NG>::kCtas))
paged_attention_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map, AttnArgs a) {
    pdl_wait();  // the dependents are let go at the CTA's last piece end, below
    using S = Shape<T, STORE, DP, NG>;
    extern __shared__ __align__(16) unsigned char s_raw[];
    unsigned char* ring = s_raw + ((1024u - (smem_addr(s_raw) & 1023u)) & 1023u);
    float* s_scales = reinterpret_cast<float*>(ring + S::kRing);          // [warp][stage][2][16]
    float* s_ml = s_scales + S::kScales / 4;                               // [warp][head][2]
    Entry* s_entry = reinterpret_cast<Entry*>(s_ml + S::kMl / 4);          // [warp][stage]
    uint64_t* s_bar = reinterpret_cast<uint64_t*>(s_entry + kWarps * S::kStages);
    Walk& walk = reinterpret_cast<Walk*>(s_bar + kWarps * S::kStages)[threadIdx.x >> 5];
    int* s_flag = reinterpret_cast<int*>(reinterpret_cast<Walk*>(s_bar + kWarps * S::kStages) + kWarps);
    int* s_slot = s_flag + 4;  // [warp]: stage of its current piece end

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = lane >> 2, col = lane & 3;  // fragment coordinates
    const int grid = gridDim.x, cta = blockIdx.x;
    const bool listed = a.list_counts != nullptr;
    const int segs = listed ? a.batch * a.kv_heads : a.batch;
    const int reps = listed ? a.head_groups : a.kv_heads * a.head_groups;
    Entry* entries = s_entry + warp * S::kStages;
    uint64_t* bars = s_bar + warp * S::kStages;
    const uint32_t ring_addr = smem_addr(ring) + warp * S::kStages * S::kBufBytes;  // this warp's buffers
    float* scales = s_scales + warp * S::kStages * 2 * kUnit;
    if (lane == 0) {
        for (int s = 0; s < S::kStages; ++s) mbar_init(&bars[s], cta == a.lost_cta ? 2 : 1);
        fence_mbar_init();
        if (warp == 0) {
            prefetch_map(&key_map);
            prefetch_map(&value_map);
        }
    }
    __syncwarp();

    const int own_units = segs <= 32 && lane < segs ? segment_units(a, lane) : 0;
    const Schedule sched = plan(a, segs, reps, own_units, lane, grid);
    Producer p;
    // The item that holds place cta * q of the line.
    int found = -1;
    {
        const int64_t lo = static_cast<int64_t>(cta) * sched.q;
        int64_t before = 0;
        int units = own_units;
        for (int s0 = 0; s0 < segs && found < 0; s0 += 32) {
            if (segs > 32) units = s0 + lane < segs ? segment_units(a, s0 + lane) : 0;
            const int64_t mine = static_cast<int64_t>(room(units, sched)) * reps;
            int64_t incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                if (o >= segs) break;
                const int64_t y = __shfl_up_sync(kFull, incl, o);
                if (lane >= o) incl += y;
            }
            const uint32_t hit = __ballot_sync(kFull, before + incl > lo);
            if (hit) {
                const int at = __ffs(hit) - 1;
                found = s0 + at;
                before += __shfl_sync(kFull, incl - mine, at);
                units = __shfl_sync(kFull, units, at);
            } else {
                before += __shfl_sync(kFull, incl, 31);
            }
        }
        if (found >= 0) {
            Walk w;
            w.seg = found;
            w.item_units = units;
            const int size = room(units, sched);
            const int64_t into = lo - before;
            w.rep = into < 0x7fffffff ? static_cast<int>(static_cast<unsigned>(into) / static_cast<unsigned>(size))
                                      : static_cast<int>(into / size);
            w.virt = before + static_cast<int64_t>(w.rep) * size + sched.gap;
            w.u0 = static_cast<int>(lo - w.virt);  // negative inside the gap
            w.left = sched.q;
            w.turn = 0;
            if (lane == 0) walk = w;
            __syncwarp();
        }
        p.done = found < 0;
    }
    // Sets the piece up that starts at walk.u0; collective.
    auto open_piece = [&]() {
        Walk w = walk;
        if (w.u0 < 0) {  // the item's gap
            w.left += w.u0;
            w.u0 = 0;
        }
        const int take = w.left < w.item_units - w.u0 ? w.left : w.item_units - w.u0;  // may be negative: only a gap
        p.end = w.u0 + take;
        // Lane i's unit is base + kWarps * i; the first look-ahead steps base forward.
        p.base = w.u0 + ((warp - w.turn) & (kWarps - 1)) - kWarps * 32;
        p.live = 0u;
        p.fresh = true;
        p.item = w.seg * reps + w.rep;
        p.b = listed ? w.seg / a.kv_heads : w.seg;
        p.kvh = listed ? w.seg - p.b * a.kv_heads : w.rep / a.head_groups;
        p.len = seq_length(a, p.b);
        __syncwarp();
        if (lane == 0) {
            walk.u0 = w.u0;
            walk.left = w.left - (sched.gap ? take : w.left);
            walk.turn = (w.turn + (take > 0 ? take : 0)) & (kWarps - 1);
        }
        __syncwarp();
        return take > 0;
    };
    if (!p.done) p.done = !open_piece();
    const bool idle = p.done;

    // Items without units: zeros, whoever's turn it is.
    for (int seg = cta; seg < segs; seg += grid) {
        if (segment_units(a, seg) != 0) continue;
        const int b = listed ? seg / a.kv_heads : seg;
        const int h0 = listed ? (seg - b * a.kv_heads) * a.G : 0, nh = listed ? a.G : a.q_heads;
        const int64_t first = static_cast<int64_t>(b) * a.q_heads + h0;
        T* o = static_cast<T*>(a.out) + first * a.head_dim;
        for (int i = threadIdx.x; i < nh * a.head_dim; i += kThreads) o[i] = from_float<T>(0.0f);
        if (a.lse != nullptr) for (int i = threadIdx.x; i < nh; i += kThreads) a.lse[first + i] = -INFINITY;
    }
    if (idle) return;

    int lost = 0;  // waits that ran out.  After the first: no further loads or barrier phases, only ends of pieces
    // Page numbers of this warp's next 32 units.  For whole sequences the table entries of the
    // 32 after them are asked for at once, so that only a piece's first look-ahead waits.
    auto look_ahead = [&](bool first) {
        const int u = p.base + kWarps * lane;
        const int upp = a.page_size / kUnit;
        const int i = upp == 1 ? u : static_cast<int>(static_cast<unsigned>(u) / static_cast<unsigned>(upp));
        const int32_t* columns = a.table + p.b * a.table_stride;
        int page = -1, column = i;
        p.info = 0;
        p.heads = kFull;
        if (listed) {
            if (u < p.end) {
                const int64_t at = (static_cast<int64_t>(p.b) * a.kv_heads + p.kvh) * a.list_capacity + i;
                column = a.list_pages[at];
                p.heads = a.list_heads[at] >> (p.item % a.head_groups * a.heads_per_item);
                if (column >= 0 && column < a.table_width) page = columns[column];
            }
        } else {
            page = first ? (u < p.end ? columns[i] : -1) : p.next_page;
            const int u2 = u + kWarps * 32;
            p.next_page = u2 < p.end ? columns[upp == 1 ? u2 : static_cast<int>(static_cast<unsigned>(u2) / static_cast<unsigned>(upp))] : -1;
        }
        if (page >= 0 && page < a.pages) {
            const int slot = (u - i * upp) * kUnit;
            const int64_t tokens = p.len - (static_cast<int64_t>(column) * a.page_size + slot);
            p.info = slot | (tokens < kUnit ? (tokens > 0 ? static_cast<int>(tokens) : 0) : kUnit) << 16;
        }
        p.page = page;
        p.live = __ballot_sync(kFull, (p.info >> 16) > 0);
    };
    // Fills stage s with this warp's next unit or piece end.
    auto push = [&](int s) {
        if (p.done) return;
        while (p.live == 0u) {
            p.base += kWarps * 32;
            if (p.base < p.end) {
                look_ahead(p.fresh);
                p.fresh = false;
                continue;
            }
            Walk w = walk;
            const int item = p.item;
            const int64_t v0 = w.virt, v1 = w.virt + w.item_units - 1;
            const bool small = v1 < 0x7fffffff;
            const int first = small ? static_cast<int>(static_cast<unsigned>(v0) / static_cast<unsigned>(sched.q)) : static_cast<int>(v0 / sched.q);
            const int last = small ? static_cast<int>(static_cast<unsigned>(v1) / static_cast<unsigned>(sched.q)) : static_cast<int>(v1 / sched.q);
            // The next item, if the share reaches into it.
            p.done = w.left <= 0;
            if (!p.done) {
                w.virt += w.item_units + sched.gap;
                w.u0 = -sched.gap;
                if (++w.rep == reps) {
                    w.rep = 0;
                    do ++w.seg; while (w.seg < segs && segment_units(a, w.seg) == 0);
                    if (w.seg < segs) w.item_units = segment_units(a, w.seg);
                }
                p.done = w.seg >= segs;
            }
            __syncwarp();
            if (lane == 0) walk = w;
            __syncwarp();
            if (!p.done) p.done = !open_piece();
            if (lost > 0) p.base = p.end;  // no unit of the next piece either
            if (lane == 0) {
                entries[s] = Entry{p.done ? -1 : 0, static_cast<uint32_t>(first), item, last};
                if (lost == 0) mbar_arrive(&bars[s]);
            }
            return;
        }
        const int k = __ffs(p.live) - 1;
        p.live &= p.live - 1u;
        if (lane == k) {  // the lane that holds the page issues the loads
            entries[s] = Entry{p.info >> 16, p.heads, p.item, 0};
            const int slot = p.info & 0xffff;
            const uint32_t buf = ring_addr + s * S::kBufBytes;
            mbar_expect_tx(&bars[s], S::kBufBytes + S::kScaleBytes);
#pragma unroll
            for (int x = 0; x < S::kBoxes; ++x)
                tma_load_4d(buf + x * kUnit * S::kBoxBytes, &key_map, x * S::kBoxChannels, slot, p.kvh, p.page, &bars[s]);
#pragma unroll
            for (int x = 0; x < S::kBoxes; ++x)
                tma_load_4d(buf + S::kPoolBytes + x * kUnit * S::kBoxBytes, &value_map, x * S::kBoxChannels, slot, p.kvh,
                            p.page, &bars[s]);
            if constexpr (S::kCached == 1) {
                const int64_t at = (static_cast<int64_t>(p.page) * a.kv_heads + p.kvh) * a.page_size + slot;
                float* sc = scales + s * 2 * kUnit;
                bulk_load(sc, a.key_scale + at, kUnit * 4, &bars[s]);
                bulk_load(sc + kUnit, a.value_scale + at, kUnit * 4, &bars[s]);
            }
        }
    };
    const int first_item = p.item;
#pragma unroll
    for (int s = 0; s < S::kStages; ++s) push(s);

    // ------------------------------------------------------------ per-piece state
    // Fragment columns: this lane's heads of group g are 8 g + 2 col + {0, 1}.
    uint32_t qf[NG][S::kSteps][2];
    float q_scale[NG][2];  // logit scales (8-bit caches)
    float acc[NG][S::kTiles][4], m[NG][2], l[NG][2], n[NG][2];
    int item = -1;
    uint32_t heads_all = 0u;  // bits of the item's heads
    auto reset = [&]() {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            m[g][0] = m[g][1] = n[g][0] = n[g][1] = -INFINITY;
            l[g][0] = l[g][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < S::kTiles; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[g][i][e] = 0.0f;
        }
    };
    // Queries of the item as B fragments (lane: head `row`), in the channel order of the K fragments.
    auto load_queries = [&]() {
        const int hg = item % a.head_groups;
        const int bk = item / a.head_groups;
        const int b = bk / a.kv_heads, kvh = bk - b * a.kv_heads;
        const int g0 = hg * a.heads_per_item;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int h = g0 + g * 8 + row;
            const bool live = g * 8 + row < a.heads_per_item && h < a.G;
            const T* q = static_cast<const T*>(a.q) + (static_cast<int64_t>(b) * a.q_heads + kvh * a.G + h) * a.head_dim;
            if constexpr (S::kCached == 2) {
#pragma unroll
                for (int x = 0; x < S::kSteps; ++x)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int ch = 16 * x + 8 * r + 2 * col;
                        uint32_t w = 0u;
                        if (live && ch < a.head_dim) {
                            const unsigned short* p2 = reinterpret_cast<const unsigned short*>(q + ch);
                            w = a.q_vec ? *reinterpret_cast<const uint32_t*>(p2) : p2[0] | static_cast<uint32_t>(p2[1]) << 16;
                        }
                        qf[g][x][r] = w;
                    }
            } else {
                constexpr int kChunks = DP / 64;  // runs of 16 channels per lane
                float top = 0.0f, up = 1.0f, scale = a.sl2;
#pragma unroll
                for (int pass = 0; pass < 2; ++pass) {
                    if (pass == 1) {
                        top = quad_max(top);
                        // 2^x brings top into [2^14, 2^15): fp16's subnormals then start at 2^-28 of it, and bf16
                        // elements, of 8 bits, are whole down to 2^-31 of it.  A head of zeros, infinities or NaN stays as it is.
                        const int biased_exponent = static_cast<int>(__float_as_uint(top) >> 23);
                        if (top > 0.0f && biased_exponent < 255) {
                            const int x = min(14 + 127 - biased_exponent, 126);
                            up = __uint_as_float(static_cast<uint32_t>(127 + x) << 23);
                            scale = a.sl2 * __uint_as_float(static_cast<uint32_t>(127 - x) << 23);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < kChunks; ++x) {
                        const int ch = DP == 64 ? 16 * col : (x >> 1) * 128 + 16 * (2 * col + (x & 1));
                        if (live && ch < a.head_dim) {
                            float f[2][8];
                            load8<T>(f[0], q + ch, a.q_vec);
                            load8<T>(f[1], q + ch + 8, a.q_vec);
#pragma unroll
                            for (int w = 0; w < 8; ++w) {
                                const float f0 = f[w >> 2][2 * (w & 3)], f1 = f[w >> 2][2 * (w & 3) + 1];
                                if (pass == 0)
                                    top = fmaxf(top, fmaxf(fabsf(f0), fabsf(f1)));
                                else
                                    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(qf[g][4 * x + (w >> 1)][w & 1]) : "f"(f1 * up), "f"(f0 * up));
                            }
                        } else if (pass == 1) {
#pragma unroll
                            for (int w = 0; w < 4; ++w) qf[g][4 * x + w][0] = qf[g][4 * x + w][1] = 0u;
                        }
                    }
                }
                q_scale[g][0] = __shfl_sync(kFull, scale, 8 * col);
                q_scale[g][1] = __shfl_sync(kFull, scale, 8 * col + 4);
            }
        }
    };

    // One unit.  FULL: 16 tokens that every head of the item attends.  Integer codes are finite whatever a
    // slot holds, so a weight of 0 is all that a masked one needs; other values are kept away from the sums.
    auto compute = [&](auto full_tag, uint32_t buf, uint32_t sc, int tokens, uint32_t heads) {
        constexpr bool FULL = decltype(full_tag)::value;
        constexpr bool GUARD = !FULL && STORE != POPKV_STORE_INT8;
        const uint32_t vbuf = buf + S::kPoolBytes;
        // Logits (base 2): s[g][0, 1] token `row`, s[g][2, 3] token row + 8, of heads 2 col + {0, 1}.
        float s[NG][4];
        {
            float c[NG][2][4];  // two chains
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) c[g][0][e] = c[g][1][e] = 0.0f;
            if constexpr (S::kCached == 2) {
                const int r = (lane & 7) + 8 * ((lane >> 3) & 1);
#pragma unroll
                for (int x = 0; x < S::kSteps; ++x) {
                    uint32_t k[4];
                    const int chunk = (2 * x & 7) + (lane >> 4);
                    ldsm4(k, buf + (x >> 2) * kUnit * 128 + r * 128 + ((chunk ^ (r & 7)) << 4));
#pragma unroll
                    for (int g = 0; g < NG; ++g)
                        mma16816<S::kBf16>(c[g][x & 1], k[0], k[1], k[2], k[3], qf[g][x][0], qf[g][x][1]);
                }
            } else {
#pragma unroll
                for (int x = 0; x < DP / 64; ++x) {
                    uint32_t k[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = row + 8 * h;
                        const uint32_t at = DP == 64 ? buf + r * 64 + ((col ^ ((r >> 1) & 3)) << 4)
                                                     : buf + (x >> 1) * kUnit * 128 + r * 128 + (((2 * col + (x & 1)) ^ (r & 7)) << 4);
                        const uint4 w = lds128(at);
                        k[h][0] = biased<STORE>(w.x); k[h][1] = biased<STORE>(w.y);
                        k[h][2] = biased<STORE>(w.z); k[h][3] = biased<STORE>(w.w);
                    }
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t a0 = codes_to_half2<STORE, false>(k[0][w]), a1 = codes_to_half2<STORE, false>(k[1][w]);
                        const uint32_t a2 = codes_to_half2<STORE, true>(k[0][w]), a3 = codes_to_half2<STORE, true>(k[1][w]);
#pragma unroll
                        for (int g = 0; g < NG; ++g)
                            mma16816<false>(c[g][w & 1], a0, a1, a2, a3, qf[g][4 * x + w][0], qf[g][4 * x + w][1]);
                    }
                }
            }
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[g][e] = c[g][0][e] + c[g][1][e];
        }
        float lv[2] = {0.0f, 0.0f};  // log2 of the tokens' value scales
        if constexpr (S::kCached == 1) {
            const float k0 = lds32f(sc + row * 4), k1 = lds32f(sc + (row + 8) * 4);
            lv[0] = lg2(lds32f(sc + (kUnit + row) * 4));
            lv[1] = lg2(lds32f(sc + (kUnit + row + 8) * 4));
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                s[g][0] *= k0 * q_scale[g][0];
                s[g][1] *= k0 * q_scale[g][1];
                s[g][2] *= k1 * q_scale[g][0];
                s[g][3] *= k1 * q_scale[g][1];
            }
        } else {
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[g][e] *= a.sl2;
        }
        bool act[NG][2];
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int e = 0; e < 2; ++e) act[g][e] = FULL || ((heads >> (8 * g + 2 * col + e)) & 1u);
        if constexpr (!FULL) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const bool in = row + 8 * t < tokens;
                if (!in) lv[t] = 0.0f;
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (!in || !act[g][e]) s[g][2 * t + e] = -INFINITY;
            }
        }
        // Weights are relative to references m (softmax sum) and n (8-bit caches: weights with value
        // scales) that only follow the running maxima once these are 2^kSlack above: most
        // units neither reduce a maximum nor touch the sums.
        [[maybe_unused]] float lw[NG][4];
        bool over = false;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                over = over || s[g][e] > m[g][e & 1] + S::kSlack;
                if constexpr (S::kCached == 1) {
                    lw[g][e] = !FULL && s[g][e] == -INFINITY ? -INFINITY : s[g][e] + lv[e >> 1];
                    over = over || lw[g][e] > n[g][e & 1] + S::kSlack;
                }
            }
        if (__any_sync(kFull, over)) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float shrink[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mn = fmaxf(m[g][e], column_max(fmaxf(s[g][e], s[g][e + 2])));
                    const float am = ex2(m[g][e] - (mn == -INFINITY ? 0.0f : mn));
                    m[g][e] = mn;
                    l[g][e] *= am;
                    shrink[e] = am;
                    if constexpr (S::kCached == 1) {
                        const float nn = fmaxf(n[g][e], column_max(fmaxf(lw[g][e], lw[g][e + 2])));
                        shrink[e] = ex2(n[g][e] - (nn == -INFINITY ? 0.0f : nn));
                        n[g][e] = nn;
                    }
                }
#pragma unroll
                for (int i = 0; i < S::kTiles; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[g][i][e] *= shrink[e & 1];
            }
        }
        uint32_t hi[NG][2], lo[NG][2];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float base = m[g][e & 1] == -INFINITY ? 0.0f : m[g][e & 1];
                if constexpr (S::kCached == 2) {
                    w[e] = ex2(s[g][e] - (base - S::kUp));
                    l[g][e & 1] += w[e];
                } else {
                    l[g][e & 1] += ex2(s[g][e] - base);
                    w[e] = ex2(lw[g][e] - ((n[g][e & 1] == -INFINITY ? 0.0f : n[g][e & 1]) - S::kUp));
                }
            }
            split_pair<S::kBf16>(w[0], w[1], hi[g][0], lo[g][0]);
            split_pair<S::kBf16>(w[2], w[3], hi[g][1], lo[g][1]);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                hi[g][t] = turn8x8(hi[g][t]);
                lo[g][t] = turn8x8(lo[g][t]);
            }
        }
        // Masked tokens' values may be anything: their bits are cleared.
        uint32_t keep0 = kFull, keep1 = kFull;
        if constexpr (GUARD) {
            keep0 = (2 * col < tokens ? 0xffffu : 0u) | (2 * col + 1 < tokens ? 0xffff0000u : 0u);
            keep1 = (2 * col + 8 < tokens ? 0xffffu : 0u) | (2 * col + 9 < tokens ? 0xffff0000u : 0u);
        }
        auto weigh = [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
            if constexpr (GUARD) {
                a0 &= keep0; a1 &= keep0;
                a2 &= keep1; a3 &= keep1;
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if constexpr (!GUARD) {
                    mma16816<S::kBf16>(acc[g][i], a0, a1, a2, a3, hi[g][0], hi[g][1]);
                    mma16816<S::kBf16>(acc[g][i], a0, a1, a2, a3, lo[g][0], lo[g][1]);
                } else {
                    // A head that does not attend the page keeps its sum: 0 times an infinity must not reach it.
                    float t[4] = {acc[g][i][0], acc[g][i][1], acc[g][i][2], acc[g][i][3]};
                    mma16816<S::kBf16>(t, a0, a1, a2, a3, hi[g][0], hi[g][1]);
                    mma16816<S::kBf16>(t, a0, a1, a2, a3, lo[g][0], lo[g][1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[g][i][e] = act[g][e & 1] ? t[e] : acc[g][i][e];
                }
            }
        };
        if constexpr (S::kCached == 2) {
            // Transposed 8x8 blocks: (channels 0-7, tokens 0-7), (8-15, 0-7), (0-7, 8-15), (8-15, 8-15).
            const int r = (lane & 7) + 8 * (lane >> 4);
#pragma unroll
            for (int i = 0; i < S::kTiles; ++i) {
                uint32_t v[4];
                const int chunk = (2 * i & 7) + ((lane >> 3) & 1);
                ldsm4t(v, vbuf + (i >> 2) * kUnit * 128 + r * 128 + ((chunk ^ (r & 7)) << 4));
                weigh(i, v[0], v[1], v[2], v[3]);
            }
        } else {
            // Bytes of 16 (DP 64: 8) channels of tokens 2 col + {0, 1, 8, 9}, paired by token: channel j of the
            // run and j + half of it make a tile's rows.
            constexpr int kHalf = DP == 64 ? 1 : 2;  // words in half a run
#pragma unroll
            for (int x = 0; x < S::kBoxes; ++x) {
                uint32_t v[4][2 * kHalf];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const int r = 2 * col + (t & 1) + 8 * (t >> 1);
                    if constexpr (DP == 64) {
                        const uint2 w = lds64(vbuf + r * 64 + (((row >> 1) ^ ((r >> 1) & 3)) << 4) + (row & 1) * 8);
                        v[t][0] = w.x; v[t][1] = w.y;
                    } else {
                        const uint4 w = lds128(vbuf + x * kUnit * 128 + r * 128 + ((row ^ (r & 7)) << 4));
                        v[t][0] = w.x; v[t][1] = w.y; v[t][2] = w.z; v[t][3] = w.w;
                    }
                }
#pragma unroll
                for (int w = 0; w < kHalf; ++w)
#pragma unroll
                    for (int p2 = 0; p2 < 2; ++p2) {  // bytes 0, 1, then 2, 3 of the words
                        const int sel = p2 ? 0x7362 : 0x5140;
                        const uint32_t b0 = biased<STORE>(__byte_perm(v[0][w], v[1][w], sel));
                        const uint32_t b1 = biased<STORE>(__byte_perm(v[0][w + kHalf], v[1][w + kHalf], sel));
                        const uint32_t b2 = biased<STORE>(__byte_perm(v[2][w], v[3][w], sel));
                        const uint32_t b3 = biased<STORE>(__byte_perm(v[2][w + kHalf], v[3][w + kHalf], sel));
                        const int i = x * 4 * kHalf + 4 * w + 2 * p2;
                        weigh(i, codes_to_half2<STORE, false>(b0), codes_to_half2<STORE, false>(b1),
                              codes_to_half2<STORE, false>(b2), codes_to_half2<STORE, false>(b3));
                        weigh(i + 1, codes_to_half2<STORE, true>(b0), codes_to_half2<STORE, true>(b1),
                              codes_to_half2<STORE, true>(b2), codes_to_half2<STORE, true>(b3));
                    }
            }
        }
    };

    // Channel of elements 0, 1 (half 0) or 2, 3 (half 1) of tile i; their heads are 2 col + {0, 1}.
    auto channel = [&](int i, int half) {
        if constexpr (S::kCached == 2) return 16 * i + 8 * half + row;
        constexpr int kRun = DP == 64 ? 8 : 16;
        return (i / (kRun / 2)) * 128 + kRun * row + i % (kRun / 2) + half * (kRun / 2);
    };
    // Channels ch .. ch + 3 of a head's output.  Nothing attended: zeros; a sum of NaN stays.
    auto write4 = [&](T* dst, int ch, const float4& x, float sum) {
        if (ch >= a.head_dim) return;  // head_dim is a multiple of 16
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        const bool none = sum == 0.0f;
        const uint32_t u = pack2<T>(none ? 0.0f : x.x * inv, none ? 0.0f : x.y * inv);
        const uint32_t v = pack2<T>(none ? 0.0f : x.z * inv, none ? 0.0f : x.w * inv);
        if (a.out_vec) {
            *reinterpret_cast<uint2*>(dst + ch) = make_uint2(u, v);
        } else {
            const unsigned short b[4] = {static_cast<unsigned short>(u), static_cast<unsigned short>(u >> 16),
                                         static_cast<unsigned short>(v), static_cast<unsigned short>(v >> 16)};
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<unsigned short*>(dst)[ch + i] = b[i];
        }
    };
    // End of a piece.  The warps' sums meet in the unit buffers of the pieces' ends, which hold no
    // unit; then a warp per head writes the piece out or leaves it as a partial ([head][channel] sums, then
    // (m, l) per head), and the CTA with the item's last ticket merges.
    auto flush = [&](const Entry& en, int at) {
        const int first = static_cast<int>(en.heads), last = en.last;
        const int hg = en.item % a.head_groups, bk = en.item / a.head_groups;
        const int left = a.G - hg * a.heads_per_item;
        const int heads = left < a.heads_per_item ? left : a.heads_per_item;
        // First query head's row of the item: heads of a KV head are neighbours.
        const int64_t out_row = static_cast<int64_t>(bk / a.kv_heads) * a.q_heads + (bk % a.kv_heads) * a.G + hg * a.heads_per_item;
        T* out = static_cast<T*>(a.out) + out_row * a.head_dim;
        float* part = a.parts + static_cast<int64_t>(2 * cta + (cta == first ? 1 : 0)) * a.part_floats;
        constexpr int kQuads = DP / 128 > 0 ? DP / 128 : 1;  // runs of 4 channels per lane
        const bool on = 4 * lane < DP;
        if (lane == 0) s_slot[warp] = at;
        // Channel c of head h sits at c ^ 8 (h / 2 % 4): no bank conflicts on the 16-bit path's stores.
        float* mine = reinterpret_cast<float*>(ring + (warp * S::kStages + at) * S::kBufBytes);
        auto sums_of = [&](int v) { return reinterpret_cast<const float*>(ring + (v * S::kStages + s_slot[v]) * S::kBufBytes); };
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float f[2], f2[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                l[g][e] = column_sum(l[g][e]);
                // Both sums in units of 2^unit.  At 16 bits they are: of 2^(m - kUp).  With 8-bit caches the
                // weights went against n, and 2^(m + kSlack) keeps the common unit above every weight.
                float unit = m[g][e] - S::kUp;
                f[e] = f2[e] = 1.0f;
                if constexpr (S::kCached == 1) {
                    unit = m[g][e] + S::kSlack;
                    l[g][e] *= ex2(-S::kSlack);
                    const float x = m[g][e] == -INFINITY || n[g][e] == -INFINITY ? 0.0f : n[g][e] - S::kUp - unit;
                    f[e] = f2[e] = ex2(0.5f * x);
                }
                // Tokens are missing: the piece's heads come out as NaN, whatever the buffers hold.
                if (lost > 0) l[g][e] = __uint_as_float(0x7fffffffu);
                if (row == 0) {
                    s_ml[(warp * S::kHeads + g * 8 + 2 * col + e) * 2] = unit;
                    s_ml[(warp * S::kHeads + g * 8 + 2 * col + e) * 2 + 1] = l[g][e];
                }
            }
            if (g > 0) __syncthreads();  // the group before this one has been read
#pragma unroll
            for (int i = 0; i < S::kTiles; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (lost == 0) mine[(2 * col + (e & 1)) * DP + (channel(i, e >> 1) ^ (8 * col))] = acc[g][i][e] * f[e & 1] * f2[e & 1];
            __syncthreads();
#pragma unroll 1
            for (int h = warp; h < 8 && g * 8 + h < heads; h += kWarps) {
                const int hd = g * 8 + h;
                float w[kWarps], base = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int v = 0; v < kWarps; ++v) {
                    w[v] = s_ml[(v * S::kHeads + hd) * 2];
                    base = fmaxf(base, w[v]);
                }
                const float ref = base == -INFINITY ? 0.0f : base;
#pragma unroll
                for (int v = 0; v < kWarps; ++v) {
                    w[v] = ex2(w[v] - ref);
                    sum += w[v] * s_ml[(v * S::kHeads + hd) * 2 + 1];
                }
                if (on) {
#pragma unroll
                    for (int k = 0; k < kQuads; ++k) {
                        const int ch = 128 * k + 4 * lane;
                        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                        for (int v = 0; v < kWarps; ++v) {
                            const float4 y = *reinterpret_cast<const float4*>(sums_of(v) + h * DP + (ch ^ (8 * ((h >> 1) & 3))));
                            x.x += w[v] * y.x; x.y += w[v] * y.y; x.z += w[v] * y.z; x.w += w[v] * y.w;
                        }
                        if (first != last) __stcg(reinterpret_cast<float4*>(part + hd * DP + ch), x);
                        else write4(out + hd * a.head_dim, ch, x, sum);
                    }
                }
                if (lane == 0) {
                    if (first != last) __stcg(reinterpret_cast<float2*>(part + S::kHeads * DP + 2 * hd), make_float2(base, sum));
                    else if (a.lse != nullptr) a.lse[out_row + hd] = sum == 0.0f ? -INFINITY : (base + lg2(sum)) * kLn2;
                }
            }
        }
        // The buffers go back to the asynchronous loads.
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        if (first == last) return;
        // The ticket releases the block's sums and acquires those of the others (the barriers around it
        // carry the other threads' accesses).
        if (threadIdx.x == 0) {
            uint32_t t;
            asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(t) : "l"(a.tickets + en.item) : "memory");
            const bool all = t == static_cast<uint32_t>(last - first);
            if (all) a.tickets[en.item] = 0u;  // every piece has taken its ticket
            *s_flag = all;
        }
        __syncthreads();
        if (*s_flag == 0) return;
        // A warp per head, a lane per 4 channels; (m, l) of 32 pieces in one load, kBatch pieces' sums
        // in flight.  Short code on purpose: it runs once a launch, from a cold instruction cache.
        constexpr int kBatch = 16 / kQuads;
        const int64_t stride = 2 * static_cast<int64_t>(a.part_floats);
#pragma unroll 1
        for (int h = warp; h < heads; h += kWarps) {
            float top = -INFINITY, sum = 0.0f, w = 0.0f;
            float4 x[kQuads];
#pragma unroll
            for (int k = 0; k < kQuads; ++k) x[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            // Partial of CTA c: slot 2 c, of the item's first CTA 2 c + 1.
            const float* src = a.parts + first * stride + a.part_floats + h * DP + 4 * lane;
#pragma unroll 1
            for (int c0 = first; c0 <= last; c0 += kBatch) {
                const bool fresh = ((c0 - first) & 31) == 0;
                float2 ml = make_float2(-INFINITY, 0.0f);
                if (fresh && c0 + lane <= last)
                    ml = __ldcg(reinterpret_cast<const float2*>(a.parts + (c0 + lane) * stride + (c0 + lane == first ? a.part_floats : 0) +
                                                                S::kHeads * DP + 2 * h));
                float4 v[kBatch][kQuads];
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
#pragma unroll
                    for (int k = 0; k < kQuads; ++k)
                        v[j][k] = c0 + j <= last && on ? __ldcg(reinterpret_cast<const float4*>(src + 128 * k))
                                                       : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    src += c0 + j == first ? stride - a.part_floats : stride;
                }
                if (fresh) {  // weights of the next 32 pieces, while the sums are on their way
                    float mx = ml.x, part_sum;
#pragma unroll
                    for (int o2 = 16; o2 > 0; o2 >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, o2));
                    mx = fmaxf(mx, top);
                    const float ref = mx == -INFINITY ? 0.0f : mx;
                    const float grow = ex2(top - ref);
                    top = mx;
                    w = ex2(ml.x - ref);
                    part_sum = w * ml.y;
#pragma unroll
                    for (int o2 = 16; o2 > 0; o2 >>= 1) part_sum += __shfl_xor_sync(kFull, part_sum, o2);
                    sum = sum * grow + part_sum;
#pragma unroll
                    for (int k = 0; k < kQuads; ++k) { x[k].x *= grow; x[k].y *= grow; x[k].z *= grow; x[k].w *= grow; }
                }
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const float wj = __shfl_sync(kFull, w, (c0 - first + j) & 31);
#pragma unroll
                    for (int k = 0; k < kQuads; ++k) {
                        x[k].x += wj * v[j][k].x; x[k].y += wj * v[j][k].y;
                        x[k].z += wj * v[j][k].z; x[k].w += wj * v[j][k].w;
                    }
                }
            }
            if (on) {
#pragma unroll
                for (int k = 0; k < kQuads; ++k) write4(out + h * a.head_dim, 128 * k + 4 * lane, x[k], sum);
            }
            if (lane == 0 && a.lse != nullptr) a.lse[out_row + h] = sum == 0.0f ? -INFINITY : (top + lg2(sum)) * kLn2;
        }
    };

    // ------------------------------------------------------------------ main loop
    reset();
    // The first item's queries arrive while its first units do.
    item = first_item;
    heads_all = item_heads(a, item);
    load_queries();
    int stage = 0;
    uint32_t parity = 0;
    for (;;) {
        // The entry was written by one lane a ring's length ago; the wait below also orders it.  What happened before is only
        // looked at off the path on which the copy has landed (ahead of every wait it cost the 8-bit caches 1.7 %).
        __syncwarp();
        const bool landed = mbar_try_wait(&bars[stage], parity) ||
                            (lost < S::kStages &&
                             mbar_wait_bounded(&bars[stage], parity, lost ? a.wait_ns / S::kStages : a.wait_ns));
        if (!__all_sync(kFull, landed)) {
            // A copy never completed: recorded.  What is in the ring is waited for a little longer, so that the shared memory is
            // not left to late copies; then the rest runs without loads and waits, so that every ticket is taken.
            if (lost == 0) {
                if (lane == 0) atomicAdd(a.tickets + kMaxItems, 1u);
                p.live = 0u;
                p.base = p.end;
            }
            ++lost;
        }
        const Entry en = entries[stage];
        if (en.tokens > 0) {
            if (lost == 0 && en.item != item) {
                item = en.item;
                heads_all = item_heads(a, item);
                load_queries();
            }
            if (lost == 0) {
                const uint32_t buf = ring_addr + stage * S::kBufBytes;
                const uint32_t sc = smem_addr(scales) + stage * 2 * kUnit * 4;
                if (STORE != POPKV_STORE_INT8 && en.tokens == kUnit && (~en.heads & heads_all) == 0u)
                    compute(std::true_type{}, buf, sc, kUnit, kFull);
                else
                    compute(std::false_type{}, buf, sc, en.tokens, en.heads);
            }
        } else {
            // Dependents may take the SM from here on.  Let go at the start, their blocks fill what this grid
            // leaves free on some SMs and sit there: page-sparse 8 x 131072, whose next kernel is the
            // scorer, took 178 us instead of 158.
            if (en.tokens < 0) pdl_trigger();
            flush(en, stage);
            if (en.tokens < 0) break;
            reset();
            item = -1;
        }
        __syncwarp();  // every lane has read the stage
        push(stage);
        if (++stage == S::kStages) {
            stage = 0;
            parity ^= 1u;
        }
    }
}

// --------------------------------------------------------------------- host side
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

// Pool [pages][kv_heads][page_size][head_dim] in boxes of [16 slots x box_bytes]; channels past head_dim read as zeros.
bool pool_map(CUtensorMap* map, const popkv_paged_cache* c, void* pool, int box_bytes) {
    const EncodeTiledFn enc = encode_tiled();
    if (enc == nullptr) return false;
    const cuuint64_t es = c->store == POPKV_STORE_SAME ? 2 : 1;
    const CUtensorMapDataType dt = es == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : c->dtype == POPKV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t dims[4] = {(cuuint64_t)c->head_dim, (cuuint64_t)c->page_size, (cuuint64_t)c->kv_heads, (cuuint64_t)c->pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c->slot_stride * es, (cuuint64_t)c->head_stride * es, (cuuint64_t)c->page_stride * es};
    const cuuint32_t box[4] = {(cuuint32_t)(box_bytes / (int)es), (cuuint32_t)kUnit, 1u, 1u};
    const cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
    return enc(map, dt, 4, pool, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int heads_per_item(int64_t G, int64_t head_dim) { return G <= 8 || head_dim > 128 ? 8 : kMaxHeads; }

// Partials of the largest grid: 2 per CTA, at most 4 CTAs per SM.
int64_t part_floats(int heads, int64_t head_dim) {
    const int64_t dp = head_dim <= 64 ? 64 : (head_dim <= 128 ? 128 : 256);
    return heads * (dp + 2);
}

// What popkv_paged_attention_lose_copies set.
std::atomic<int> g_lost_cta{-1};
std::atomic<unsigned long long> g_wait_ns{kWaitNs};

template <typename T, int STORE, int DP, int NG>
int launch(const popkv_paged_cache* cache, const AttnArgs& a, cudaStream_t st) {
    using S = Shape<T, STORE, DP, NG>;
    CUtensorMap km, vm;
    if (!pool_map(&km, cache, cache->keys, S::kBoxBytes) || !pool_map(&vm, cache, cache->values, S::kBoxBytes))
        return fail(POPKV_ERR_UNSUPPORTED, "no tensor map for this paged cache");
    auto kern = paged_attention_kernel<T, STORE, DP, NG>;
    static bool sized[64] = {};  // per device; setting it twice is harmless
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = -1;
    if (dev < 0 || !sized[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess)
            return check_launch("popkv_paged_attention");
        if (dev >= 0) sized[dev] = true;
    }
    launch_pdl(kern, dim3((unsigned)(num_sms() * S::kCtas)), dim3(kThreads), S::kSmem, st, km, vm, a);
    return check_launch("popkv_paged_attention");
}

template <typename T, int STORE>
int launch_dim(const popkv_paged_cache* cache, const AttnArgs& a, cudaStream_t st) {
    const bool wide = a.heads_per_item > 8;
    if (cache->head_dim > 128) return launch<T, STORE, 256, 1>(cache, a, st);
    if (cache->head_dim > 64) return wide ? launch<T, STORE, 128, 2>(cache, a, st) : launch<T, STORE, 128, 1>(cache, a, st);
    return wide ? launch<T, STORE, 64, 2>(cache, a, st) : launch<T, STORE, 64, 1>(cache, a, st);
}

}  // namespace
}  // namespace popkv

using namespace popkv;

extern "C" size_t popkv_paged_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
    if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || head_dim <= 0) return 0;
    return (size_t)(kTicketBytes + 2 * 4 * (int64_t)num_sms() * part_floats(heads_per_item(q_heads / kv_heads, head_dim), head_dim) * 4);
}

extern "C" void popkv_paged_attention_lose_copies(int64_t block, uint64_t limit_ns) {
    g_lost_cta.store(block < 0 || block > 0x7fffffff ? -1 : (int)block, std::memory_order_relaxed);
    g_wait_ns.store(limit_ns == 0 || limit_ns > kWaitNs ? kWaitNs : limit_ns, std::memory_order_relaxed);
}

extern "C" int popkv_paged_attention(const void* q, const popkv_paged_cache* cache, const int32_t* table,
                                     int64_t table_stride, int64_t table_width, const int32_t* lengths, int64_t batch,
                                     int64_t q_heads, float scale, const popkv_page_list* list, void* out, float* lse,
                                     void* workspace, size_t workspace_bytes, popkv_stream_t stream) {
    if (const int rc = check_paged_cache(cache)) return rc;
    if (batch < 0 || q_heads <= 0 || q_heads % cache->kv_heads || table_width < 0 || table_width > 0x7fffffffLL / 1024 ||
        (batch > 1 && table_stride < table_width))
        return fail(POPKV_ERR_INVALID_ARGUMENT, "invalid paged attention shape");
    if (batch == 0) return POPKV_OK;
    const int64_t G = q_heads / cache->kv_heads;
    const int per_item = heads_per_item(G, cache->head_dim);
    const int64_t groups = (G + per_item - 1) / per_item;
    if (batch > kMaxItems || cache->kv_heads * groups > kMaxItems || batch * cache->kv_heads * groups > kMaxItems)
        return fail(POPKV_ERR_UNSUPPORTED, "too many heads and sequences for one call");
    if (!q || !out || !lengths || !workspace || (table_width > 0 && !table))
        return fail(POPKV_ERR_INVALID_ARGUMENT, "null pointer argument");
    if (!aligned(workspace, 16)) return fail(POPKV_ERR_ALIGNMENT, "workspace needs 16-byte alignment");
    if (list && (!list->counts || list->capacity < 0 || (list->capacity > 0 && (!list->pages || !list->heads)) || G > 32))
        return fail(POPKV_ERR_INVALID_ARGUMENT, "invalid page list");
    if (list && list->capacity > (1 << 26) / (cache->page_size / 16))
        return fail(POPKV_ERR_UNSUPPORTED, "page list of more than 2^30 tokens");
    if (workspace_bytes < popkv_paged_workspace_bytes(batch, q_heads, cache->kv_heads, cache->head_dim))
        return fail(POPKV_ERR_WORKSPACE, "paged attention workspace too small");
    AttnArgs a = {};
    a.q = q; a.out = out; a.lse = lse;
    a.key_scale = cache->key_scale; a.value_scale = cache->value_scale;
    a.pages = cache->pages;
    a.table = table; a.table_stride = table_stride; a.table_width = (int)table_width;
    a.lengths = lengths;
    a.batch = (int)batch; a.q_heads = (int)q_heads; a.kv_heads = (int)cache->kv_heads; a.G = (int)G;
    a.head_groups = (int)groups; a.heads_per_item = per_item;
    a.head_dim = (int)cache->head_dim; a.page_size = (int)cache->page_size;
    a.sl2 = scale * kLog2e;
    a.q_vec = aligned(q, 16);
    a.out_vec = aligned(out, 8);
    if (list) {
        a.list_pages = list->pages; a.list_heads = list->heads; a.list_counts = list->counts;
        a.list_capacity = list->capacity;
    }
    a.tickets = static_cast<uint32_t*>(workspace);
    a.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + kTicketBytes);
    a.part_floats = (int)part_floats(per_item, cache->head_dim);
    a.lost_cta = g_lost_cta.load(std::memory_order_relaxed);
    a.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
    const cudaStream_t st = as_stream(stream);
    auto by = [&](auto* tp) {
        using T = std::remove_pointer_t<decltype(tp)>;
        switch (cache->store) {
            case POPKV_STORE_INT8: return launch_dim<T, POPKV_STORE_INT8>(cache, a, st);
            case POPKV_STORE_E4M3: return launch_dim<T, POPKV_STORE_E4M3>(cache, a, st);
            default: return launch_dim<T, POPKV_STORE_SAME>(cache, a, st);
        }
    };
    return cache->dtype == POPKV_BF16 ? by(static_cast<__nv_bfloat16*>(nullptr)) : by(static_cast<__half*>(nullptr));
}
