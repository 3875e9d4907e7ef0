// emb_paged_attend: attention of one new token of each request over the pages of a cache.
//
//   out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s_j = scale log2(e) q . k_j,  m = max_j s_j
//
// One pass over the keys with the running maximum and sum of the softmax: when a key raises the maximum from m to m', what
// was summed is scaled by 2^(m - m'). Every key and value is read once for the heads / kv_heads query heads that share it,
// so the bound is HBM: 2 dim bytes of cache per 2 * group * dim multiply-adds of each product.
//
// Products are mma.sync m16n8k16 with the KEYS as rows: S^T = K Q^T (16 keys x 8 query heads) and O^T = V^T P^T (16 dims x
// 8 heads), so a group of up to eight heads wastes no row, and S^T becomes the operand P^T by one 8 x 8 transposition
// (movmatrix). tcgen05 would want 128 rows of one request and head at a time in shared memory as it lays them out; the
// tensor work here is a seventh of what the legacy path does in the time HBM needs for the bytes. A WARP owns KEYS
// consecutive keys at a time: it copies them into a ring of its own with cp.async (rows found through the page table, so any
// page size and any strides; rows behind the length are filled with zeros and not read), multiplies, and keeps a maximum,
// sum and output of its own. No barrier stands between copies and products.
// The warps of a CTA either take the keys of one head in turn (a tile is WARPS * KEYS keys), and meet at the head's end, or,
// where there is enough work and the number of heads allows, stand SIDE BY SIDE on neighbouring heads (a tile is KEYS keys of
// each): then no warp waits for another, and a token's rows of several heads are read at about the same time.
// What weights refer to moves only when a score passes the maximum it came from by more than 8: most steps then need neither the
// reduction over lanes nor the rescaling. For products of f16 it lies 7 below that maximum: a weight is at most 2^15, still below
// f16's largest number, and the least that is not 0 is 2^-32 of the row's largest weight. (With the maximum itself it was 2^-25:
// of 131072 keys that all have 2^-25.2 of the leading one's weight, 0.3 % of the result was lost.)
// A weight is two 16-bit numbers and so two products with the values (`split`). One alone is off by as much as the result's own
// rounding: the mean error against 64 bits was 1.3 times that of a result rounded once. The second product costs under 1 %
// where HBM is the bound (8 x 4096 keys 87.6 -> 88.1, 64 ragged requests 168.1 -> 168.8 us), 4 % over e4m3 codes with f16 queries
// and 8 to 13 % with 16 query heads and more of 128 a key head (64 requests up to 4000 keys: 57.5 -> 62.3 us with 64 on 4 key
// heads, 48.1 -> 54.3 with 64 on 2), whatever the order of the products.
//
// The work is cut by TILES, all requests and heads (or sets of heads side by side) behind one another: CTA c of n takes
// tiles [c T / n, (c + 1) T / n), whatever their requests. So a single long request and a ragged batch both spread evenly, and
// a request's head is cut only where a CTA's share ends. Those pieces (maximum, sum, unscaled output; two per CTA at
// most) go to the workspace, and paged_join_kernel adds them up in the order of the keys.
//
// Measured (a pass among others, join included; of the measured copy rate of 6.55 TB/s): 8 requests x 4096 keys x 32 key heads
// of 128, f16, 537 MB: 88 us, 0.93 (the kernel alone 83 us, 0.99); 64 ragged requests up to 8192 keys, 32 query heads on 8 key
// heads, bf16, 1070 MB: 169 us, 0.97; one request of 131072 keys, 537 MB: 90 us, 0.91; 128 requests of up to 2000 keys, 64
// query heads on 8 key heads of 64, e4m3, 224 MB: 55 us, 0.62 (the codes' decode and a row's bookkeeping: 46 % of the issue slots,
// with three warps a scheduler to fill them; rows of 64 bytes come at 5 to 6.3 TB/s whatever reads them). Small calls are bound
// by latency: 6.2 us for one request of 113 keys, 8 where pieces are joined.
// Farther from one reading of the bytes (us, and us at the copy rate): groups of more than eight query heads (62 / 38: 64 requests
// up to 4000 keys, 64 on 4 heads of 128), e4m3 of 128 and 256 (52 / 38, 38 / 19), calls of 10 to 150 MB (30 / 18: 56 requests up
// to 8000 keys, one key head of 128; about 8 us are fixed), many requests of few keys at 256 dims (13: 115 of 2 keys, 5 heads).

#include "paged_common.cuh"

#include <algorithm>
#include <atomic>
#include <optional>

#include "emb_frag.cuh"

namespace {

using namespace emb::paged;
namespace frag = emb::frag;

// Where no request can have more than about so many keys, and there are no more tiles than CTAs, heads are not cut and
// nothing is joined: four requests of 240 keys take 7.5 us so and 8.3 cut (128 dims, bf16), two of 900 keys 10.1 and 8.9 (64
// dims, e4m3).
constexpr int WHOLE_KEYS = 256;
// Warps stand side by side where there are at least SIDE_SETS sets of heads for every 100 CTAs (a head is then spread over
// few CTAs, and the join is short) and a CTA gets at least SIDE_TILES tiles (below, the latency of a head's keys one after
// another counts, and they are better shared by the warps).
constexpr int SIDE_SETS = 12, SIDE_TILES = 8;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

constexpr float LOWEST = -3.402823466e38f;  // seed of a maximum: finite, so that a masked score (-inf) against it weighs 0
constexpr float SLACK = 8.f;  // log2 of how far a score may pass the maximum that what weights refer to came from

template <class T, class C, int DIM_, int HT_> struct Config {
    static constexpr int DIM = DIM_, HT = HT_, ROWS = 8 * HT;  // query heads of a CTA, in tiles of eight
    static constexpr bool CODES = sizeof(C) == 1;
    static constexpr bool BF16 = !CODES && std::is_same<T, __nv_bfloat16>::value;  // type of the products
    static constexpr float BELOW = BF16 ? 0.f : 7.f;  // log2: what weights refer to, below the maximum
    // whether a weight is held as two 16-bit numbers: where one would be off by as much as the result's own rounding is. (Over
    // e4m3 codes the products are of f16, whose steps are an eighth of a bf16 result's; to split there too took 54 -> 57 us, 128
    // requests of 2000 keys, 64-wide heads.)
    static constexpr bool SPLIT = BF16 || std::is_same<T, __half>::value;
    static constexpr int ROW_BYTES = DIM * static_cast<int>(sizeof(C));
    static constexpr int KEYS = ROW_BYTES >= 256 ? 16 : ROW_BYTES == 128 ? 32 : 64;  // of a warp per step
    static constexpr int STEP_BYTES = 2 * KEYS * ROW_BYTES;                         // keys, then values
    // three CTAs with two steps of 8 KB a warp were faster than two with three: 86 against 98 us (64 requests up to 4000 keys,
    // 8 key heads of 128, bf16), and than four or five with steps of half the keys (53 against 66 us, e4m3). Two steps in flight
    // before the first wait instead of one were 2 to 3 % slower
    static constexpr int WARPS = ROW_BYTES == 512 ? 2 : 4, THREADS = WARPS * 32;
    static constexpr int CTAS = 3;                                                  // per SM
    static constexpr int TILE = WARPS * KEYS;                                       // where the warps share a head
    static constexpr int TILE_SHIFT = (KEYS == 64 ? 6 : KEYS == 32 ? 5 : 4) + (WARPS == 4 ? 2 : 1);
    static_assert(TILE == 1 << TILE_SHIFT, "a power of two");
    static constexpr int PITCH = DIM + 4;         // floats of a row of a piece: outputs, maximum, sum
    static constexpr int MERGED = 512 / DIM;      // query heads whose parts the warps merge at a time
    static constexpr int MERGE_BYTES = WARPS * MERGED * PITCH * 4;
    static constexpr int STAGES = (228 * 1024 / CTAS - 1024 - 128 - MERGE_BYTES) / (WARPS * STEP_BYTES);
    static constexpr int SMEM = WARPS * STAGES * STEP_BYTES + MERGE_BYTES;
    static_assert(STAGES >= 2, "a step is copied while another is multiplied");
    static_assert(CTAS * (SMEM + 1024 + 128) <= 228 * 1024, "shared memory of an SM");
};

// A head that was cut: the CTA that holds its first tiles, how many hold one (0: nothing to join), and the warp's place
// beside the others. A CTA has two places for pieces for each warp: of the head that an earlier CTA began, and of the head
// that goes on in later ones. A list has `side` records for each CTA (of the heads that go on), or one for each head where
// those are fewer.
struct Record {
    int32_t request, head, cta, pieces, slot, unused[3];
};
struct Places {  // of records and pieces
    Record* records;
    float* pieces;  // null: no head is cut
    int32_t by_head, side, floats;  // heads side by side at most; floats of a piece
    __device__ __forceinline__ float* piece(long long cta, int second, int slot) const { return pieces + ((2 * cta + second) * side + slot) * floats; }
};

struct Heads {  // how query heads fall on the rows of a CTA
    int group, groups, cut;  // query heads of a key head; row groups they make; cut heads of a request
    __host__ __device__ Heads(const emb_paged_attend_t& a, int rows) {
        group = a.heads / a.cache.kv_heads;
        groups = (group + rows - 1) / rows;
        cut = a.cache.kv_heads * groups;
    }
};

struct Span {
    uint32_t begin, end;  // keys of a request that are attended
};

__device__ __forceinline__ Span span_of(const emb_paged_attend_t& a, int b) {
    const uint32_t capacity = static_cast<uint32_t>(a.table_width) * a.cache.page_size;
    // (a length beyond the table row keeps one key that has no page, which gives NaN)
    const uint32_t n = min(static_cast<uint32_t>(max(a.lengths[b], 0)), capacity + 1);
    return {a.window && n > a.window ? n - a.window : 0u, n};
}

// tiles begin at a multiple of 16 keys, at or before the first one
__device__ __forceinline__ uint32_t tiles_of(const Span& s, int shift) { return max(1u, (s.end - (s.begin & ~15u) + (1u << shift) - 1) >> shift); }

struct Cursor {  // a tile of the CTA's share
    int b, set;  // heads side by side: set * side + the warp's place
    uint32_t t, tiles;
    Span span;
};

__device__ __forceinline__ void advance(Cursor& c, const emb_paged_attend_t& a, int sets, int shift) {
    if (++c.t < c.tiles) return;
    c.t = 0;
    if (++c.set < sets) return;
    c.set = 0;
    if (++c.b >= a.requests) return;
    c.span = span_of(a, c.b);
    c.tiles = tiles_of(c.span, shift);
}


// A copy brings 128 bytes into L2 unless it says otherwise. A row of 64 bytes (64 e4m3 codes) of a token-major cache has
// another head's row beside it, read at another time: 64 bytes of each 128 were fetched at 3.4 TB/s of useful bytes
// without the hint and at 6.1 with it.
template <int ROW_BYTES> __device__ __forceinline__ void copy16(uint32_t to, const void* from) {
    if (ROW_BYTES == 64)
        asm volatile("cp.async.cg.shared.global.L2::64B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else if (ROW_BYTES == 128)
        asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else
        asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void fill16(uint32_t to, uint32_t word) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to), "r"(word) : "memory");
}

template <int ROW_BYTES> __device__ __forceinline__ uint32_t place(int row, int chunk) {  // of a 16-byte chunk: eight rows' equal chunks in eight bank groups
    return row * ROW_BYTES + ((chunk ^ (ROW_BYTES >= 128 ? row & 7 : (row >> 1) & 3)) << 4);
}

__device__ __forceinline__ void load4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// four e4m3 codes -> two pairs of f16, exact
__device__ __forceinline__ void widen4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
    asm("{.reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(lo), "=r"(hi) : "r"(codes));
}
__device__ __forceinline__ float exp2_(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// one more part of a row: its outputs and sum, scaled by f to the common maximum
__device__ __forceinline__ void add_part(float4& acc, float& s, const float4& x, float f, float sum) {
    acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
    s += f * sum;
}

// what a finished row's sum of weighted values is multiplied with; a row without keys is 0
template <class Cfg> __device__ __forceinline__ float share_of(const emb_paged_attend_t& a, float s) { return s == 0.f ? 0.f : (Cfg::CODES ? a.cache.v_scale : 1.f) / s; }
__device__ __forceinline__ float log_sum(float top, float s) { return s == 0.f ? -INFINITY : top * LN2 + logf(s); }

// four dims of a finished row, rounded once
template <class Cfg, class T> __device__ __forceinline__ void put_out(const emb_paged_attend_t& a, int b, long long h, int d, const float4& acc, float best, float s) {
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    const float inv = share_of<Cfg>(a, s);
    const uint2 packed = make_uint2(frag::pack_f32<BF16>(acc.x * inv, acc.y * inv), frag::pack_f32<BF16>(acc.z * inv, acc.w * inv));
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + b * a.out_stride[0] + h * a.out_stride[1] + d) = packed;
    if (a.lse && d == 0) a.lse[b * static_cast<long long>(a.heads) + h] = log_sum(best, s);
}

// P^T of eight keys: from rows of keys (a lane: key g, heads 2 quad, 2 quad + 1) to the operand (keys 2 quad, 2 quad + 1, head g)
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Two weights as one operand and what is left of them as another. The first parts are cut off a little below the weights, so
// that what is left is never 0 beside a weight that is not: an infinite value stays infinite (0 * inf would be NaN).
// Together they are off by at most 2^-20 of a weight (f16; 2^-25 where that is more) or 2^-14 (bf16).
template <bool BF16> __device__ __forceinline__ void split(float u, float v, uint32_t& first, uint32_t& left) {
    if (BF16) {
        const uint32_t a = __float_as_uint(u * (1.f - 0x1p-7f)), b = __float_as_uint(v * (1.f - 0x1p-7f));
        first = __byte_perm(a, b, 0x7632);
        left = frag::pack_f32<true>(u - __uint_as_float(a & 0xffff0000u), v - __uint_as_float(b & 0xffff0000u));
    } else {
        const float a = fmaxf(fmaf(u, 1.f - 0x1p-10f, -0x1p-24f), 0.f), b = fmaxf(fmaf(v, 1.f - 0x1p-10f, -0x1p-24f), 0.f);
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(first) : "f"(b), "f"(a));
        const float2 x = __half22float2(reinterpret_cast<const __half2&>(first));
        left = frag::pack_f32<false>(u - x.x, v - x.y);
    }
}

template <class T, class C, int DIM, int HT>
__global__ void __launch_bounds__((Config<T, C, DIM, HT>::THREADS), (Config<T, C, DIM, HT>::CTAS)) paged_attend_kernel(const __grid_constant__ emb_paged_attend_t a, const Divisor page_size, const Places places) {
    using Cfg = Config<T, C, DIM, HT>;
    constexpr int WARPS = Cfg::WARPS, THREADS = Cfg::THREADS, KEYS = Cfg::KEYS, KT = KEYS / 16, DT = DIM / 16, ROW_BYTES = Cfg::ROW_BYTES, STAGES = Cfg::STAGES;
    constexpr int LOOKS = (KEYS + 31) / 32;  // keys that a lane looks up per step, at most
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ long long scan_slab[2][WARPS], share[2];
    __shared__ uint32_t first_tile;
    __shared__ int first_request, first_set, holders;  // the share's first tile; holders: CTAs from this one on that hold tiles of the head its share ends in
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, quad = lane & 3;
    follow_on();
    const Heads heads(a, Cfg::ROWS);
    const bool lists = places.pieces && !places.by_head;  // this CTA owes `side` records

    // ---- how the warps stand, and the CTA's share of the tiles
    const int side_shift = Cfg::TILE_SHIFT - (places.side >= 4 ? 2 : places.side >= 2 ? 1 : 0);
    // tiles of the requests up to and with base + tid of this pass, in either way, and of all in the pass
    const auto scan = [&](int base, const Span& s, long long& in_turn, long long& beside, long long (&sums)[2]) {
        const bool real = base + tid < a.requests;
        in_turn = real ? static_cast<long long>(tiles_of(s, Cfg::TILE_SHIFT)) * heads.cut : 0;
        beside = real ? static_cast<long long>(tiles_of(s, side_shift)) * (heads.cut / places.side) : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, in_turn, d), y = __shfl_up_sync(0xffffffffu, beside, d);
            if (lane >= d) in_turn += x, beside += y;
        }
        if (base) __syncthreads();  // the slab's last readers are done
        if (lane == 31) scan_slab[0][warp] = in_turn, scan_slab[1][warp] = beside;
        __syncthreads();
        sums[0] = sums[1] = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) in_turn += scan_slab[0][w], beside += scan_slab[1][w];
            sums[0] += scan_slab[0][w], sums[1] += scan_slab[1][w];
        }
    };
    Span span = tid < a.requests ? span_of(a, tid) : Span{0, 0};
    long long in_turn, beside, sums[2], totals[2];
    scan(0, span, in_turn, beside, totals);
    for (int base = THREADS; base < a.requests; base += THREADS) {
        long long x, y;
        scan(base, base + tid < a.requests ? span_of(a, base + tid) : Span{0, 0}, x, y, sums);
        totals[0] += sums[0], totals[1] += sums[1];
    }
    const bool stand = totals[1] >= static_cast<long long>(SIDE_TILES) * gridDim.x && static_cast<long long>(a.requests) * (heads.cut / places.side) * 100 >= SIDE_SETS * static_cast<long long>(gridDim.x);
    const int side = stand ? places.side : 1;
    const int sharing = WARPS / side;  // warps on one head
    const int shift = side > 1 ? side_shift : Cfg::TILE_SHIFT, sets = heads.cut / side;
    const int slot = warp / sharing, turn_of = warp % sharing;  // the warp's head in a set, and its turn among those on it
    const long long all = side > 1 ? totals[1] : totals[0];
    const long long n = min(static_cast<long long>(gridDim.x), all);
    if (static_cast<long long>(blockIdx.x) >= n) {
        if (tid < places.side && lists) places.records[blockIdx.x * places.side + tid].pieces = 0;
        return;
    }
    const bool whole = !places.pieces;  // no place for pieces: no cuts
    const auto border = [&](uint32_t c) {  // all c / n; a 64-bit division takes longer than all else here
        return all * (c + 1ll) < (1ll << 32) ? static_cast<long long>(static_cast<uint32_t>(all * c) / static_cast<uint32_t>(n)) : all * c / n;
    };
    const long long want0 = border(blockIdx.x), want1 = border(blockIdx.x + 1);
    if (tid == 0) share[0] = want0, share[1] = want1, holders = 0;
    __syncthreads();
    long long before_pass = 0;
    for (int base = 0; base < a.requests; base += THREADS) {
        if (a.requests > THREADS) {  // (else the first scan's sums are at hand)
            span = base + tid < a.requests ? span_of(a, base + tid) : Span{0, 0};
            __syncthreads();
            scan(base, span, in_turn, beside, sums);
        }
        const uint32_t tiles = base + tid < a.requests ? tiles_of(span, shift) : 0u;
        const long long upto = before_pass + (side > 1 ? beside : in_turn), from = upto - static_cast<long long>(tiles) * sets;
        if (a.requests > THREADS) before_pass += side > 1 ? sums[1] : sums[0];
        // a border inside a head that is not to be cut moves to the head's first tile
        if (from <= want0 && want0 < upto) {
            const uint32_t ahead_of = static_cast<uint32_t>(want0 - from);  // (a request's tiles of all heads are fewer than 2^32)
            const uint32_t set = ahead_of / tiles, t = whole ? 0 : ahead_of - set * tiles;
            share[0] = from + static_cast<long long>(set) * tiles + t;
            first_request = base + tid, first_set = set, first_tile = t;
        }
        if (from <= want1 && want1 < upto) {
            const long long head_from = from + static_cast<long long>(static_cast<uint32_t>(want1 - from) / tiles) * tiles;
            if (whole) share[1] = head_from;
            else if (head_from < want1) holders = static_cast<int>(((head_from + tiles) * n + all - 1) / all - blockIdx.x);
        }
    }
    __syncthreads();
    const long long x0 = share[0], x1 = share[1];
    if (x0 >= x1) {
        if (tid < places.side && lists) places.records[blockIdx.x * places.side + tid].pieces = 0;
        return;
    }
    Cursor ahead;
    ahead.b = first_request;
    ahead.span = span_of(a, ahead.b);
    ahead.tiles = tiles_of(ahead.span, shift);
    ahead.set = first_set;
    ahead.t = first_tile;
    Cursor now = ahead;
    const auto token_at = [&](const Cursor& c) { return (c.span.begin & ~15u) + (c.t << shift) + turn_of * KEYS; };  // the warp's first

    // ---- copies: a lane finds a key's row, the warp copies KEYS of them
    const uint32_t ring = frag::smem_addr(smem) + warp * (STAGES * Cfg::STEP_BYTES);
    const uint32_t k_stride[3] = {static_cast<uint32_t>(a.cache.k_stride[0]), static_cast<uint32_t>(a.cache.k_stride[1]), static_cast<uint32_t>(a.cache.k_stride[2])};
    const uint32_t v_stride[3] = {static_cast<uint32_t>(a.cache.v_stride[0]), static_cast<uint32_t>(a.cache.v_stride[1]), static_cast<uint32_t>(a.cache.v_stride[2])};
    const bool same = k_stride[0] == v_stride[0] && k_stride[1] == v_stride[1] && k_stride[2] == v_stride[2];
    // where pages are multiples of 16 tokens, sixteen keys lie in one page behind one another: a lane looks up sixteen at a
    // time, else one
    const bool sixteens = page_size.d % 16 == 0;
    const auto token_of = [&](int look) {
        return token_at(ahead) + (sixteens ? lane % (KEYS / 16) * 16 : look * 32 + lane % min(KEYS, 32));
    };
    // found a step before they are needed: the page id (-1: behind the length, -2: none) and the token in it
    int page[LOOKS];
    uint32_t in_page[LOOKS];
    const auto find_pages = [&]() {
#pragma unroll
        for (int l = 0; l < LOOKS; ++l) {
            if (l && sixteens) break;
            const uint32_t token = token_of(l), index = page_size.over(token);
            in_page[l] = token - index * page_size.d;
            page[l] = -1;
            if (token < ahead.span.end && (sixteens || token >= ahead.span.begin)) {
                const uint32_t id = index < static_cast<uint32_t>(a.table_width) ? a.table[ahead.b * a.table_stride + index] : -2;
                page[l] = min(id, 0xfffffffeu);  // (an entry of -1 is a page that is not there, too)
            }
        }
    };
    constexpr int CHUNKS = ROW_BYTES / 16, PER_PASS = 32 / CHUNKS;  // 16-byte pieces of a row; rows that the warp copies at once
    const int chunk = lane % CHUNKS;
    const unsigned long long k_step = k_stride[1] * sizeof(C), v_step = v_stride[1] * sizeof(C);  // bytes from a token to the next
    const char* const k_from = static_cast<const char*>(a.cache.k) + chunk * 16;
    const char* const v_from = static_cast<const char*>(a.cache.v) + chunk * 16;
    const auto issue = [&](int stage) {
        const uint32_t kv = (ahead.set * side + slot) / heads.groups;
        // byte offsets of the rows (strides are below 2^32 elements), or the page id where there is no row
        long long k_at[LOOKS], v_at[LOOKS];
#pragma unroll
        for (int l = 0; l < LOOKS; ++l) {
            if (l && sixteens) break;
            const bool one = static_cast<uint32_t>(page[l]) < static_cast<uint32_t>(a.cache.pages);
            const unsigned long long id = static_cast<uint32_t>(page[l]);
            k_at[l] = one ? (id * k_stride[0] + static_cast<unsigned long long>(in_page[l]) * k_stride[1] + static_cast<unsigned long long>(kv) * k_stride[2]) * sizeof(C) : page[l] == -1 ? -1 : -2;
            v_at[l] = k_at[l];
            if (!same && one) v_at[l] = (id * v_stride[0] + static_cast<unsigned long long>(in_page[l]) * v_stride[1] + static_cast<unsigned long long>(kv) * v_stride[2]) * sizeof(C);
        }
        const uint32_t to = ring + stage * Cfg::STEP_BYTES;
        const uint32_t token0 = token_at(ahead);
        uint32_t rest = (1u << (KEYS / 16)) - 1;  // sixteens that are not copied whole
        if (sixteens) {
#pragma unroll
            for (int s = 0; s < KEYS / 16; ++s) {
                const long long k_first = __shfl_sync(0xffffffffu, k_at[0], s), v_first = same ? k_first : __shfl_sync(0xffffffffu, v_at[0], s);
                if (k_first < 0 || token0 + s * 16 < ahead.span.begin || token0 + s * 16 + 16 > ahead.span.end) continue;
                rest &= ~(1u << s);
                const char* k_row = k_from + k_first + (lane / CHUNKS) * k_step;
                const char* v_row = v_from + v_first + (lane / CHUNKS) * v_step;
#pragma unroll
                for (int p = 0; p < 16 / PER_PASS; ++p) {
                    const uint32_t k_to = to + place<ROW_BYTES>(s * 16 + p * PER_PASS + lane / CHUNKS, chunk);
                    copy16<ROW_BYTES>(k_to, k_row);
                    copy16<ROW_BYTES>(k_to + KEYS * ROW_BYTES, v_row);
                    k_row += k_step * PER_PASS, v_row += v_step * PER_PASS;
                }
            }
        }
        if (!rest) return;
        // row by row: the ends of a span, pages that are not there, pages of other sizes
#pragma unroll 1
        for (int p = 0; p < KEYS / PER_PASS; ++p) {
            if (!(rest >> (p * PER_PASS / 16) & 1)) continue;
            const int row = p * PER_PASS + lane / CHUNKS, source = sixteens ? row >> 4 : row & 31;
            const bool second = LOOKS > 1 && !sixteens && row >= 32;
            long long k_row = __shfl_sync(0xffffffffu, k_at[0], source), v_row = __shfl_sync(0xffffffffu, v_at[0], source);
            if (LOOKS > 1) {
                const long long k_other = __shfl_sync(0xffffffffu, k_at[LOOKS - 1], source), v_other = __shfl_sync(0xffffffffu, v_at[LOOKS - 1], source);
                if (second) k_row = k_other, v_row = v_other;
            }
            if (token0 + row < ahead.span.begin || token0 + row >= ahead.span.end) k_row = -1;
            const uint32_t k_to = to + place<ROW_BYTES>(row, chunk), v_to = k_to + KEYS * ROW_BYTES;
            if (k_row >= 0) {
                const unsigned long long in = sixteens ? row & 15 : 0;
                copy16<ROW_BYTES>(k_to, k_from + k_row + in * k_step);
                copy16<ROW_BYTES>(v_to, v_from + v_row + in * v_step);
            } else {  // not attended: zeros; no such page: keys of NaN
                fill16(k_to, k_row == -1 ? 0u : Cfg::CODES ? 0x7f7f7f7fu : 0x7fff7fffu);
                fill16(v_to, 0u);
            }
        }
    };

    const uint32_t steps = static_cast<uint32_t>(x1 - x0);
    uint32_t issued = 0;
    find_pages();
    const auto feed = [&](int stage) {
        if (issued < steps) {
            issue(stage);
            advance(ahead, a, sets, shift);
            if (issued + 1 < steps) find_pages();
        }
        ++issued;
        frag::cp_async_commit();
    };
    for (int s = 0; s < STAGES - 1; ++s) feed(s);

    uint32_t q[HT][DT][2];
    float factor[HT][2];                  // of the products of heads 2 quad and 2 quad + 1: into score log2(e)
    float top[HT][2], total[HT][2];       // what their weights refer to; this lane's keys' part of the sum
    float o[HT][DT][4];                   // dims g and g + 8 of 16 (codes: 2 g and 2 g + 1), heads 2 quad and 2 quad + 1
    // a negative scale turns the query's signs, and scale 0 is a query of 0: so the largest product is the largest score
    // (and a scale that underflows stays above 0: a masked score is -inf and not -inf * 0)
    const float scale = a.scale == 0.f ? 1.f : fmaxf(fabsf(a.scale) * LOG2E * (Cfg::CODES ? a.cache.k_scale : 1.f), 1.2e-38f);
    const uint32_t turn = a.scale < 0.f ? 0x80008000u : 0u;
    // the query rows of the head that comes next: loaded before the last one's parts are merged, used behind that (behind it
    // where the registers would not hold both)
    constexpr bool EARLY = !Cfg::CODES || DIM * HT <= 128;
    uint2 raw[Cfg::CODES ? HT : 1][Cfg::CODES ? DT : 1];
    const auto load_queries = [&]() {
        const int head = now.set * side + slot, kv = head / heads.groups, row0 = (head % heads.groups) * Cfg::ROWS;
#pragma unroll
        for (int m = 0; m < HT; ++m) {
            const int row = row0 + m * 8 + g;
            const T* from = static_cast<const T*>(a.q) + now.b * a.q_stride[0] + (static_cast<long long>(kv) * heads.group + row) * a.q_stride[1];
            const bool real = row < heads.group && a.scale != 0.f;
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                if (Cfg::CODES) {
                    raw[m][d] = real ? *reinterpret_cast<const uint2*>(from + d * 16 + quad * 4) : make_uint2(0u, 0u);
                } else {
                    q[m][d][0] = real ? *reinterpret_cast<const uint32_t*>(from + d * 16 + quad * 2) ^ turn : 0u;
                    q[m][d][1] = real ? *reinterpret_cast<const uint32_t*>(from + d * 16 + 8 + quad * 2) ^ turn : 0u;
                }
            }
        }
    };
    const auto begin_head = [&]() {
#pragma unroll
        for (int m = 0; m < HT; ++m) {
            float mine = scale;
            if (Cfg::CODES) {
                // an e4m3 row's dims 4 quad .. 4 quad + 3 come in one word, so the query's dims are dealt the same way. The
                // product is of f16: a bf16 query's row is first scaled by a power of two to 2^14 <= max < 2^15, the top of
                // f16's range (its 8 bits are kept down to 2^-28 of the row's maximum, and a rounding below is 2^-39 of it)
                float most = 0.f;
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const T* x = reinterpret_cast<const T*>(&raw[m][d]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(to_f32(x[e])));
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                int power = ((__float_as_int(most) >> 23) & 255) - 127;
                power = std::is_same<T, __half>::value ? 0 : max(-100, min(power, 127)) - 14;
                const float down = __int_as_float((127 - power) << 23);
                mine = fmaxf(scale * __int_as_float((127 + power) << 23), 1.2e-38f);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    const T* x = reinterpret_cast<const T*>(&raw[m][d]);
                    q[m][d][0] = frag::pack_f32<false>(to_f32(x[0]) * down, to_f32(x[1]) * down) ^ turn;
                    q[m][d][1] = frag::pack_f32<false>(to_f32(x[2]) * down, to_f32(x[3]) * down) ^ turn;
                }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                factor[m][e] = Cfg::CODES ? __shfl_sync(0xffffffffu, mine, (quad * 2 + e) * 4) : scale;
                top[m][e] = LOWEST, total[m][e] = 0.f;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[m][d][e] = 0.f;
        }
    };

    float* const merge = reinterpret_cast<float*>(smem + WARPS * STAGES * Cfg::STEP_BYTES);
    const auto meet = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + slot), "r"(sharing * 32) : "memory"); };  // of the warps on one head
    // the sums of heads 2 quad and 2 quad + 1 over the lanes' keys
    const auto sums_of = [&](int m, float (&sum)[2]) {
        sum[0] = total[m][0], sum[1] = total[m][1];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1)
#pragma unroll
            for (int e = 0; e < 2; ++e) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], d);
    };
    const auto put_part = [&](int m, int e, float sum, float* to) {  // a row's outputs, maximum and sum
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if (Cfg::CODES) *reinterpret_cast<float2*>(to + d * 16 + g * 2) = make_float2(o[m][d][e], o[m][d][e + 2]);
            else to[d * 16 + g] = o[m][d][e], to[d * 16 + g + 8] = o[m][d][e + 2];
        }
        if (g == 0) *reinterpret_cast<float2*>(to + DIM) = make_float2(top[m][e], sum);
    };
    // a head that the warp has alone: out, or to its piece
    const auto end_alone = [&](int b, int head, float* piece) {
        const int kv = head / heads.groups, row0 = (head % heads.groups) * Cfg::ROWS;
        const int rows = min(Cfg::ROWS, heads.group - row0);
#pragma unroll
        for (int m = 0; m < HT; ++m) {
            if (m * 8 >= rows) break;
            float sum[2], inv[2];
            sums_of(m, sum);
            if (piece) {
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (m * 8 + quad * 2 + e < rows) put_part(m, e, sum[e], piece + (m * 8 + quad * 2 + e) * Cfg::PITCH);
                continue;
            }
            const long long h0 = static_cast<long long>(kv) * heads.group + row0 + m * 8;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                inv[e] = share_of<Cfg>(a, sum[e]);
                if (a.lse && g == 0 && m * 8 + quad * 2 + e < rows) a.lse[b * static_cast<long long>(a.heads) + h0 + quad * 2 + e] = log_sum(top[m][e], sum[e]);
            }
            T* const to = static_cast<T*>(a.out) + b * a.out_stride[0] + (h0 + g) * a.out_stride[1];
            constexpr bool OUT_BF16 = std::is_same<T, __nv_bfloat16>::value;
#pragma unroll
            for (int d = 0; d < DT; ++d) {  // turned: a lane has dims of head g
                const uint32_t x = transposed(frag::pack_f32<OUT_BF16>(o[m][d][0] * inv[0], o[m][d][1] * inv[1]));
                const uint32_t y = transposed(frag::pack_f32<OUT_BF16>(o[m][d][2] * inv[0], o[m][d][3] * inv[1]));
                if (m * 8 + g >= rows) continue;
                if (Cfg::CODES) {  // x: dims 4 quad and 4 quad + 2, y: 4 quad + 1 and 4 quad + 3
                    *reinterpret_cast<uint2*>(to + d * 16 + quad * 4) = make_uint2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
                } else {
                    *reinterpret_cast<uint32_t*>(to + d * 16 + quad * 2) = x;
                    *reinterpret_cast<uint32_t*>(to + d * 16 + 8 + quad * 2) = y;
                }
            }
        }
    };
    // one that warps share: their maxima, sums and outputs become one, MERGED query heads at a time
    const auto end_shared = [&](int b, int head, float* piece) {
        const int kv = head / heads.groups, row0 = (head % heads.groups) * Cfg::ROWS;
        const int rows = min(Cfg::ROWS, heads.group - row0);
#pragma unroll
        for (int m = 0; m < HT; ++m) {
            if (m * 8 >= rows) break;
            float sum[2];
            sums_of(m, sum);
#pragma unroll
            for (int first = 0; first < 8; first += Cfg::MERGED) {
                if (m * 8 + first >= rows) break;
                meet();  // the last heads are read
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int r = quad * 2 + e - first;
                    if (r >= 0 && r < Cfg::MERGED && m * 8 + first + r < rows) put_part(m, e, sum[e], merge + (warp * Cfg::MERGED + r) * Cfg::PITCH);
                }
                meet();
                const float* const parts = merge + slot * sharing * Cfg::MERGED * Cfg::PITCH;
                for (int i = turn_of * 32 + lane; i < Cfg::MERGED * (DIM / 4); i += sharing * 32) {
                    const int r = i / (DIM / 4), d = i % (DIM / 4) * 4, row = m * 8 + first + r;
                    if (row >= rows) break;
                    float best = LOWEST;
#pragma unroll
                    for (int w = 0; w < WARPS; ++w)
                        if (w < sharing) best = fmaxf(best, parts[(w * Cfg::MERGED + r) * Cfg::PITCH + DIM]);
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                    float s = 0.f;
#pragma unroll
                    for (int w = 0; w < WARPS; ++w) {
                        if (w >= sharing) break;
                        const float* from = parts + (w * Cfg::MERGED + r) * Cfg::PITCH;
                        add_part(acc, s, *reinterpret_cast<const float4*>(from + d), exp2_(from[DIM] - best), from[DIM + 1]);
                    }
                    if (piece) {
                        float* to = piece + row * Cfg::PITCH;
                        *reinterpret_cast<float4*>(to + d) = acc;
                        if (d == 0) *reinterpret_cast<float2*>(to + DIM) = make_float2(best, s);
                    } else {
                        put_out<Cfg, T>(a, b, static_cast<long long>(kv) * heads.group + row0 + row, d, acc, best, s);
                    }
                }
            }
        }
    };

    load_queries();
    begin_head();
    int stage = 0;
    bool cut_in_front = now.t > 0;  // the head's tiles before these belong to an earlier CTA
    Record record{};  // of the head that goes on
    for (uint32_t step = 0; step < steps; ++step) {
        frag::cp_async_wait<STAGES - 2>();
        __syncwarp();
        feed(stage == 0 ? STAGES - 1 : stage - 1);
        const uint32_t from = ring + stage * Cfg::STEP_BYTES;
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        const uint32_t token0 = token_at(now);
        if (token0 < now.span.end) {
            // ---- scores
            constexpr int CHAINS = HT * KT >= 4 ? 1 : 2;  // sums that a score is made of: products of one sum wait for one another
            float s[HT][KT][4], s2[HT][KT][4];            // keys g and g + 8 of 16, heads 2 quad and 2 quad + 1
#pragma unroll
            for (int m = 0; m < HT; ++m)
#pragma unroll
                for (int j = 0; j < KT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[m][j][e] = s2[m][j][e] = 0.f;
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                if (!Cfg::CODES) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        uint32_t r[4];
                        load4(r, from + place<ROW_BYTES>(j * 16 + (lane & 15), d * 2 + (lane >> 4)));
#pragma unroll
                        for (int m = 0; m < HT; ++m) frag::mma_f32<Cfg::BF16>(CHAINS == 2 && d % 2 ? s2[m][j] : s[m][j], r, q[m][d]);
                    }
                } else {
#pragma unroll
                    for (int d = 0; d < DT; d += 2) {
                        uint32_t r[4];
                        load4(r, from + place<ROW_BYTES>(j * 16 + (lane & 15), d + (lane >> 4)));
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            uint32_t w[4];
                            widen4(r[2 * i], w[0], w[2]);
                            widen4(r[2 * i + 1], w[1], w[3]);
#pragma unroll
                            for (int m = 0; m < HT; ++m) frag::mma_f32<false>(CHAINS == 2 && i ? s2[m][j] : s[m][j], w, q[m][d + i]);
                        }
                    }
                }
            }

            // ---- softmax
            if (CHAINS == 2) {
#pragma unroll
                for (int m = 0; m < HT; ++m)
#pragma unroll
                    for (int j = 0; j < KT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[m][j][e] += s2[m][j][e];
            }
            if (token0 < now.span.begin || token0 + KEYS > now.span.end) {
#pragma unroll
                for (int j = 0; j < KT; ++j)
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        if (token0 + j * 16 + half * 8 + g < now.span.begin || token0 + j * 16 + half * 8 + g >= now.span.end) {
#pragma unroll
                            for (int m = 0; m < HT; ++m) s[m][j][half * 2] = s[m][j][half * 2 + 1] = -INFINITY;
                        }
            }
            float most[HT][2];
            bool passed = false;
#pragma unroll
            for (int m = 0; m < HT; ++m)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    most[m][e] = s[m][0][e];
#pragma unroll
                    for (int j = 0; j < KT; ++j)
#pragma unroll
                        for (int half = 0; half < 2; ++half) most[m][e] = fmaxf(most[m][e], s[m][j][half * 2 + e]);
                    most[m][e] *= factor[m][e];
                    passed |= most[m][e] - top[m][e] > SLACK + Cfg::BELOW;  // (exact where it is near, whatever their size)
                }
            if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
                for (int m = 0; m < HT; ++m)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = most[m][e];
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                        const float raised = fmaxf(top[m][e], x - Cfg::BELOW), keep = exp2_(top[m][e] - raised);
                        top[m][e] = raised;
                        total[m][e] *= keep;
#pragma unroll
                        for (int d = 0; d < DT; ++d) o[m][d][e] *= keep, o[m][d][e + 2] *= keep;
                    }
            }
            uint32_t p[HT][KT][2], left[HT][KT][2];  // the weights as operands
#pragma unroll
            for (int m = 0; m < HT; ++m)
#pragma unroll
                for (int j = 0; j < KT; ++j)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        // (the product is rounded as that of the maximum was: no weight passes 2^15, however large the scores)
                        const float u = exp2_(__fsub_rn(__fmul_rn(s[m][j][half * 2], factor[m][0]), top[m][0]));
                        const float v = exp2_(__fsub_rn(__fmul_rn(s[m][j][half * 2 + 1], factor[m][1]), top[m][1]));
                        total[m][0] += u, total[m][1] += v;
                        // the product with the values takes 16-bit operands (f16 or bf16)
                        if (Cfg::SPLIT) {
                            split<Cfg::BF16>(u, v, p[m][j][half], left[m][j][half]);
                            p[m][j][half] = transposed(p[m][j][half]), left[m][j][half] = transposed(left[m][j][half]);
                        } else {  // the weights' one rounding, to 2^-11
                            p[m][j][half] = transposed(frag::pack_f32<Cfg::BF16>(u, v));
                        }
                    }

            // ---- values
            const uint32_t values = from + KEYS * ROW_BYTES;
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                const int row = j * 16 + (lane & 7) + ((lane & 16) >> 1), chunk = (lane >> 3) & 1;
                if (!Cfg::CODES) {
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        uint32_t r[4];
                        load4_trans(r, values + place<ROW_BYTES>(row, d * 2 + chunk));
#pragma unroll
                        for (int m = 0; m < HT; ++m) frag::mma_f32<Cfg::BF16>(o[m][d], r, p[m][j]);
#pragma unroll
                        for (int m = 0; m < HT; ++m) frag::mma_f32<Cfg::BF16>(o[m][d], r, left[m][j]);
                    }
                } else {
#pragma unroll
                    for (int d = 0; d < DT; d += 2) {
                        uint32_t r[4];
                        load4_trans(r, values + place<ROW_BYTES>(row, d + chunk));
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            // a word holds dims (2g, 2g + 1) of two keys: sorted by dim, the even dims are the tile's first eight rows
                            uint32_t w[4];
                            widen4(__byte_perm(r[i], 0, 0x3120), w[0], w[1]);
                            widen4(__byte_perm(r[i + 2], 0, 0x3120), w[2], w[3]);
#pragma unroll
                            for (int m = 0; m < HT; ++m) frag::mma_f32<false>(o[m][d + i], w, p[m][j]);
                            if (Cfg::SPLIT) {
#pragma unroll
                                for (int m = 0; m < HT; ++m) frag::mma_f32<false>(o[m][d + i], w, left[m][j]);
                            }
                        }
                    }
                }
            }
        }

        // ---- the end of a head, or of the share
        const bool head_ends = now.t + 1 == now.tiles, share_ends = step + 1 == steps;
        const int b = now.b, head = now.set * side + slot;
        if (head_ends || share_ends) {
            float* piece = nullptr;
            if (cut_in_front || !head_ends) piece = places.piece(blockIdx.x, !cut_in_front, slot);
            if (!head_ends && !cut_in_front) record = {b, head, static_cast<int>(blockIdx.x), holders, slot, {}};  // it starts here and goes on
            if (places.by_head && turn_of == 0 && lane == 0 && !cut_in_front) places.records[b * heads.cut + head] = head_ends ? Record{} : record;
            cut_in_front = false;
            if (!share_ends) {
                advance(now, a, sets, shift);
                if (EARLY) load_queries();
            }
            if (sharing == 1) end_alone(b, head, piece);
            else end_shared(b, head, piece);
            if (!share_ends) {
                if (!EARLY) load_queries();
                begin_head();
            }
        } else {
            ++now.t;
        }
    }
    if (lists) {
        if (turn_of == 0 && lane == 0) places.records[blockIdx.x * places.side + slot] = record;
        if (tid >= side && tid < places.side) places.records[blockIdx.x * places.side + tid].pieces = 0;
    }
}

// The pieces of the heads that were cut. `split` warps (1, 2, 4 or 8) have a row of a record; its maximum and sum are joined as
// in the kernel above. The warps' parts are added in order: always the same order, so results do not depend on timing. What it
// takes is the latency of three dependent loads, if a warp has few pieces and all warps have a place at once. (A CTA for each
// record took 12.8 us with a cold L2 where 1776 of them have two pieces of four rows.)
constexpr int JOIN_WARPS = 8;

template <class T, class C, int DIM, int HT>
__global__ void __launch_bounds__(JOIN_WARPS * 32) paged_join_kernel(const __grid_constant__ emb_paged_attend_t a, const Places places, const Divisor rows, uint32_t units, int split) {
    using Cfg = Config<T, C, DIM, HT>;
    constexpr int PER_LANE = DIM / 32, BATCH = 4;  // dims of a lane; pieces loaded at a time
    __shared__ __align__(16) float slab[JOIN_WARPS][DIM + 4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % split;
    const uint32_t unit = (blockIdx.x * JOIN_WARPS + warp) / split, of = rows.over(unit);
    const int r = unit - of * rows.d;
    follow_on();
    const Heads heads(a, Cfg::ROWS);
    const Record record = unit < units ? places.records[of] : Record{};
    const int kv = record.head / heads.groups, row0 = (record.head % heads.groups) * Cfg::ROWS;
    const bool live = record.pieces > 0 && r < heads.group - row0;
    float acc[PER_LANE] = {}, s = 0.f, best = LOWEST;
    if (live) {
        // the first in its CTA's second place, the others in their CTAs' first
        const auto piece = [&](int i) -> const float* { return places.piece(record.cta + i, i == 0, record.slot) + r * Cfg::PITCH; };
        for (int k = lane; k < record.pieces; k += 32) best = fmaxf(best, piece(k)[DIM]);
        for (int k0 = part; k0 < record.pieces || k0 == part; k0 += BATCH * split) {
            float x[BATCH][PER_LANE];
            float2 stat[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const float* const p = piece(min(k0 + u * split, record.pieces - 1));
                stat[u] = *reinterpret_cast<const float2*>(p + DIM);
#pragma unroll
                for (int e = 0; e < PER_LANE; e += 2) {
                    const float2 y = *reinterpret_cast<const float2*>(p + lane * PER_LANE + e);
                    x[u][e] = y.x, x[u][e + 1] = y.y;
                }
            }
            if (k0 == part) {  // behind the first batch's loads
#pragma unroll
                for (int d = 16; d; d >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, d));
            }
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                if (k0 + u * split >= record.pieces) break;
                const float f = exp2_(stat[u].x - best);
#pragma unroll
                for (int e = 0; e < PER_LANE; ++e) acc[e] += f * x[u][e];
                s += f * stat[u].y;
            }
        }
    }
    if (split > 1) {
#pragma unroll
        for (int e = 0; e < PER_LANE; ++e) slab[warp][lane * PER_LANE + e] = acc[e];
        if (lane == 0) slab[warp][DIM] = s;
        __syncthreads();
        if (part) return;
        for (int w = 1; w < split; ++w) {
#pragma unroll
            for (int e = 0; e < PER_LANE; ++e) acc[e] += slab[warp + w][lane * PER_LANE + e];
            s += slab[warp + w][DIM];
        }
    }
    if (!live) return;
    const float inv = share_of<Cfg>(a, s);
    const long long h = static_cast<long long>(kv) * heads.group + row0 + r;
    T* const to = static_cast<T*>(a.out) + record.request * a.out_stride[0] + h * a.out_stride[1] + lane * PER_LANE;
#pragma unroll
    for (int e = 0; e < PER_LANE; e += 2) *reinterpret_cast<uint32_t*>(to + e) = frag::pack_f32<std::is_same<T, __nv_bfloat16>::value>(acc[e] * inv, acc[e + 1] * inv);
    if (a.lse && lane == 0) a.lse[record.request * static_cast<long long>(a.heads) + h] = log_sum(best, s);
}

// no request's tiles cover more keys (one without a page among them where a length is beyond its table row, and up to 15
// before a window)
int64_t longest_of(const emb_paged_attend_t& a) {
    const int64_t most = static_cast<int64_t>(a.table_width) * a.cache.page_size + 1;
    return a.window ? std::min<int64_t>(a.window + 15ll, most) : most;
}

// the CTAs of a launch: as many as the SMs hold at once, or as there can be tiles
template <class Cfg> int grid_of(const emb_paged_attend_t& a, int sms) {
    const double most = static_cast<double>(a.requests) * Heads(a, Cfg::ROWS).cut * ((longest_of(a) + Cfg::TILE - 1) / Cfg::TILE);
    const int all = sms * Cfg::CTAS;
    return most < all ? static_cast<int>(most) : all;
}

// What a call writes and reads, but for the workspace, whose bytes are known later. (out may be q: a head's queries are in
// registers before its output is written, by the CTA that has the head to itself or by the join.)
struct Memory {
    Area written[2], read[5];
    explicit Memory(const emb_paged_attend_t& a)
        : written{rows_at("out", a.out, a.requests, a.heads, a.cache.dim, a.out_stride), Area("lse", a.lse, int64_t(a.requests) * a.heads * 4)},
          read{rows_at("q", a.q, a.requests, a.heads, a.cache.dim, a.q_stride), pages_at("the keys' pages", a.cache, a.cache.k, a.cache.k_stride),
               pages_at("the values' pages", a.cache, a.cache.v, a.cache.v_stride), Area("table", a.table, int64_t(a.table_width) * 4).by(a.requests, a.table_stride * 4),
               Area("lengths", a.lengths, int64_t(a.requests) * 4)} {}
    int refuse_shared() const {
        const char* which[2];
        return touches(written, read, &read[0], which) ? refuse("paged_attend: %s and %s share memory", which[0], which[1]) : 0;
    }
    int refuse_shared(const void* workspace, int64_t bytes) const {
        const Area w[1] = {Area("the workspace", workspace, bytes)};
        const char* which[2];
        return touches(w, written, nullptr, which) || touches(w, read, nullptr, which) ? refuse("paged_attend: %s and %s share memory", which[0], which[1]) : 0;
    }
};

template <class T, class C, int DIM, int HT> int run(const emb_paged_attend_t& a, const Memory* memory, cudaStream_t stream, int64_t* need) {
    using Cfg = Config<T, C, DIM, HT>;
    const int sms = sm_count();
    if (!sms) return refuse("paged_attend: the current device cannot be asked for its SMs");
    const int grid = grid_of<Cfg>(a, sms);
    const bool cuts = grid == sms * Cfg::CTAS || longest_of(a) > std::max(WHOLE_KEYS, static_cast<int>(Cfg::TILE));  // else no head is cut
    const Heads heads(a, Cfg::ROWS);
    const int64_t cut_heads = static_cast<int64_t>(a.requests) * heads.cut;
    Places places = {};
    places.side = heads.cut % Cfg::WARPS == 0 ? Cfg::WARPS : heads.cut % 2 == 0 ? 2 : 1;
    places.by_head = cuts && cut_heads <= static_cast<int64_t>(grid) * places.side;
    places.floats = std::min(heads.group, static_cast<int>(Cfg::ROWS)) * Cfg::PITCH;
    const int64_t list = places.by_head ? cut_heads : static_cast<int64_t>(grid) * places.side;
    const int64_t bytes = cuts ? list * static_cast<int64_t>(sizeof(Record)) + 2ll * grid * places.side * places.floats * 4 : 0;
    if (need) {
        *need = bytes;
        return 0;
    }
    if (bytes && (a.workspace_bytes < bytes || !a.workspace || !aligned16(a.workspace)))
        return refuse("paged_attend: a workspace of %lld bytes (16-byte aligned) is needed, not %lld", static_cast<long long>(bytes), static_cast<long long>(a.workspace_bytes));
    if (int r = bytes ? memory->refuse_shared(a.workspace, bytes) : 0) return r;
    auto kernel = paged_attend_kernel<T, C, DIM, HT>;
    static std::atomic<bool> sized[MAX_DEVICES];  // (threads that race here set the same value)
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess) return refuse("paged_attend: no current device");
    if (!sized[device].load(std::memory_order_acquire)) {
        if (int r = launched("paged_attend's shared memory", cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM))) return r;
        sized[device].store(true, std::memory_order_release);
    }
    if (cuts) {
        places.records = static_cast<Record*>(a.workspace);
        places.pieces = reinterpret_cast<float*>(places.records + list);
    }
    if (int r = launched("launch of paged_attend", launch(kernel, dim3(grid), Cfg::THREADS, Cfg::SMEM, stream, a, Divisor(a.cache.page_size), places))) return r;
    if (!cuts) return 0;
    // as many warps for a row as have a place at once
    const int rows = std::min(heads.group, static_cast<int>(Cfg::ROWS));
    const int64_t units = list * rows, at_once = 4ll * JOIN_WARPS * sms;
    const int split = units * 8 <= at_once ? 8 : units * 4 <= at_once ? 4 : units * 2 <= at_once ? 2 : 1;
    return launched("launch of paged_join", launch(paged_join_kernel<T, C, DIM, HT>, dim3(static_cast<unsigned>((units * split + JOIN_WARPS - 1) / JOIN_WARPS)), JOIN_WARPS * 32, 0, stream, a, places,
                                                   Divisor(rows), static_cast<uint32_t>(units), split));
}

template <class T, class C> int run_dim(const emb_paged_attend_t& a, const Memory* memory, cudaStream_t stream, int64_t* need) {
    // a group of more query heads than a CTA's rows is cut into several, which read the same keys: 32 query heads of 128 in one
    // CTA need more registers than it has, and took 75 us where two of 16 took 50. Those are heads of their own in the order of
    // the tiles, a whole head apart, so unless they stand side by side HBM delivers the keys once for each: 64 requests up to
    // 4000 keys, 64 on 2 heads, take 54 us where one reading takes 19
    const int group = a.heads / a.cache.kv_heads;
    switch (a.cache.dim) {
        case 64: return group <= 8 ? run<T, C, 64, 1>(a, memory, stream, need) : run<T, C, 64, 2>(a, memory, stream, need);
        case 128: return group <= 8 ? run<T, C, 128, 1>(a, memory, stream, need) : run<T, C, 128, 2>(a, memory, stream, need);
        default: return run<T, C, 256, 1>(a, memory, stream, need);
    }
}

int attend(const emb_paged_attend_t* args, void* stream, int64_t* need) {
    if (!args) return refuse("paged_attend: null arguments");
    const emb_paged_attend_t& a = *args;
    if (int r = check_cache("paged_attend", a.cache, a.dtype)) return r;
    if (a.requests < 0 || a.heads < 1 || a.heads > 65535 || a.heads % a.cache.kv_heads)
        return refuse("paged_attend: %d requests of %d heads over %d key heads: a multiple of the key heads", a.requests, a.heads, a.cache.kv_heads);
    if (a.table_width < 1 || static_cast<int64_t>(a.table_width) * a.cache.page_size >= (1ll << 31) - 1024 || a.table_stride < 0)
        return refuse("paged_attend: a table row of %d pages of %d tokens", a.table_width, a.cache.page_size);
    if (static_cast<double>(a.table_width) * a.cache.page_size / 16 * a.heads >= 4.0e9) return refuse("paged_attend: a table row of %d pages of %d tokens for %d heads", a.table_width, a.cache.page_size, a.heads);
    if (a.window < 0) return refuse("paged_attend: a negative window");
    if (!(a.scale > -INFINITY && a.scale < INFINITY)) return refuse("paged_attend: the scale is not a finite number");
    if (need) *need = 0;
    if (a.requests == 0) return 0;
    std::optional<Memory> memory;  // (of a call for the size alone it is not looked at)
    if (!need) {
        if (!a.table || !a.lengths) return refuse("paged_attend: null table or lengths");
        if (!a.q || !a.out || !aligned16(a.q) || !aligned16(a.out)) return refuse("paged_attend: q or out is null or not 16-byte aligned");
        for (const int64_t* s : {a.q_stride, a.out_stride})
            if (!stride_fits(s[0], 2) || !stride_fits(s[1], 2)) return refuse("paged_attend: a stride of q or out is not a multiple of 16 bytes below 2^32 elements");
        const int64_t rows[2] = {a.requests, a.heads};
        if (!rows_apart(rows, a.out_stride, a.cache.dim)) return refuse("paged_attend: rows of out overlap");
        if (int r = memory.emplace(a).refuse_shared()) return r;
    }
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.dtype == EMB_F16) return a.cache.dtype == EMB_U8 ? run_dim<__half, E4m3>(a, memory ? &*memory : nullptr, s, need) : run_dim<__half, __half>(a, memory ? &*memory : nullptr, s, need);
    return a.cache.dtype == EMB_U8 ? run_dim<__nv_bfloat16, E4m3>(a, memory ? &*memory : nullptr, s, need) : run_dim<__nv_bfloat16, __nv_bfloat16>(a, memory ? &*memory : nullptr, s, need);
}

}  // namespace

extern "C" int emb_paged_attend(const emb_paged_attend_t* args, void* stream) { return attend(args, stream, nullptr); }

extern "C" int64_t emb_paged_attend_workspace(const emb_paged_attend_t* args) {
    int64_t need = 0;
    const int r = attend(args, nullptr, &need);
    return r ? (r < 0 ? r : -static_cast<int64_t>(r)) : need;
}
