// emb_paged_attend: attention of one new token of each request over the pages of a cache.
//
//   out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s_j = scale log2(e) q . k_j,  m = max_j s_j
//
// One pass over the keys with the running maximum and sum of the softmax: when a key raises the maximum from m to m', what
// was summed is scaled by 2^(m - m'). Every key and value is read once for the heads / kv_heads query heads that share it,
// so the bound is HBM: 2 dim bytes of cache per 2 * group * dim multiply-adds of each product.
//
// The group's query heads are the 16 rows (MT tiles of them) of mma.sync m16n8k16; tcgen05 would want 128 rows, and the
// tensor work of 16 rows is a tenth of what the legacy path does in the time HBM needs for the bytes. A WARP owns KEYS
// consecutive keys at a time: it copies them into a ring of its own with cp.async (rows found through the page table, so any
// page size and any strides; rows behind the length are filled with zeros and not read), multiplies, and keeps a maximum,
// sum and output of its own. Warps meet only at the end of a request's head, so no barrier stands between copies and products.
//
// The work is cut by TILES of WARPS * KEYS keys, all requests and heads behind one another: CTA c of n takes tiles
// [c T / n, (c + 1) T / n), whatever their requests. So a single long request and a ragged batch both spread evenly, and
// a request's head is cut only where a CTA's share ends. Those pieces (maximum, sum, unscaled output; two per CTA at
// most) go to the workspace, and paged_join_kernel adds them up in the order of the keys.

#include "paged_common.cuh"

#include <mutex>

#include "emb_frag.cuh"

namespace {

using namespace emb::paged;
namespace frag = emb::frag;

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int WHOLE_TILES = 4;  // a request's head of at most so many tiles is not cut
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

template <class T, class C, int DIM_, int MT_> struct Config {
    static constexpr int DIM = DIM_, MT = MT_, ROWS = 16 * MT;
    static constexpr bool CODES = sizeof(C) == 1;
    static constexpr bool BF16 = !CODES && std::is_same<T, __nv_bfloat16>::value;  // type of the products
    static constexpr int ROW_BYTES = DIM * static_cast<int>(sizeof(C));
    static constexpr int KEYS = ROW_BYTES <= 128 ? 32 : 16;  // of a warp per step
    static constexpr int TILE = WARPS * KEYS;
    static constexpr int STEP_BYTES = 2 * KEYS * ROW_BYTES;  // keys, then values
    static constexpr int CTAS = DIM == 256 ? 1 : 2;  // per SM
    static constexpr int STAGES = (192 / CTAS) * 1024 / (WARPS * STEP_BYTES);
    static constexpr int PITCH = DIM + 4;  // floats of a row of a piece: outputs, maximum, sum
    static constexpr int MERGE_BYTES = WARPS * 8 * PITCH * 4;
    static constexpr int SMEM = WARPS * STAGES * STEP_BYTES + MERGE_BYTES;
    static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory of an SM");
};

// where a piece's rows lie: the record of a CTA whose last head goes on in the next CTAs, and two pieces a CTA
struct Record {
    int32_t request, head, pieces, unused;  // head: of the cut work (key head, row group); pieces 0: nothing to join
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

template <int TILE> __device__ __forceinline__ uint32_t tiles_of(const Span& s) { return max(1u, (s.end - s.begin + TILE - 1) / TILE); }

struct Cursor {  // a tile of the CTA's share
    int b, head;
    uint32_t t, tiles;
    Span span;
};

template <class Cfg> __device__ __forceinline__ void advance(Cursor& c, const emb_paged_attend_t& a, int cut) {
    if (++c.t < c.tiles) return;
    c.t = 0;
    if (++c.head < cut) return;
    c.head = 0;
    if (++c.b >= a.requests) return;
    c.span = span_of(a, c.b);
    c.tiles = tiles_of<Cfg::TILE>(c.span);
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

template <class T, class C, int DIM, int MT>
__global__ void __launch_bounds__(THREADS, (Config<T, C, DIM, MT>::CTAS)) paged_attend_kernel(const emb_paged_attend_t a, Record* __restrict__ records, float* __restrict__ pieces) {
    using Cfg = Config<T, C, DIM, MT>;
    constexpr int KEYS = Cfg::KEYS, NT = KEYS / 8, DT = DIM / 8, ROW_BYTES = Cfg::ROW_BYTES, STAGES = Cfg::STAGES;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ long long scan_slab[WARPS], share[2];
    __shared__ long long first_before;  // tiles before the request that holds the share's first tile
    __shared__ int first_request;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, quad = lane & 3;
    follow_on();
    const Heads heads(a, Cfg::ROWS);

    // ---- the CTA's share of the tiles
    const auto scan = [&](int base, uint32_t& tiles, long long& total) -> long long {  // tiles up to and with request base + tid
        tiles = base + tid < a.requests ? tiles_of<Cfg::TILE>(span_of(a, base + tid)) : 0u;
        long long v = static_cast<long long>(tiles) * heads.cut;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += x;
        }
        __syncthreads();
        if (lane == 31) scan_slab[warp] = v;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) v += scan_slab[w];
            total += scan_slab[w];
        }
        return v;
    };
    long long all = 0, chunk_total;
    uint32_t tiles;
    long long upto = 0;
    for (int base = 0; base < a.requests; base += THREADS) {
        upto = scan(base, tiles, chunk_total) + all;
        all += chunk_total;
    }
    const long long n = min(static_cast<long long>(gridDim.x), all);
    if (static_cast<long long>(blockIdx.x) >= n) {
        if (tid == 0) records[blockIdx.x].pieces = 0;
        return;
    }
    if (tid < 2) share[tid] = all * (blockIdx.x + tid) / n;
    __syncthreads();
    const long long want0 = share[0], want1 = share[1];
    long long before_chunk = 0;
    for (int base = 0; base < a.requests; base += THREADS) {
        if (a.requests > THREADS) {
            upto = scan(base, tiles, chunk_total) + before_chunk;
            before_chunk += chunk_total;
        }
        const long long from = upto - static_cast<long long>(tiles) * heads.cut;
        // a border inside a head that is not to be cut moves to the head's first tile
        if (from <= want0 && want0 < upto) {
            const long long x = tiles <= WHOLE_TILES ? from + (want0 - from) / tiles * tiles : want0;
            share[0] = x, first_request = base + tid, first_before = from;
        }
        if (from <= want1 && want1 < upto && tiles <= WHOLE_TILES) share[1] = from + (want1 - from) / tiles * tiles;
    }
    __syncthreads();
    const long long x0 = share[0], x1 = share[1];
    if (x0 >= x1) {
        if (tid == 0) records[blockIdx.x].pieces = 0;
        return;
    }
    Cursor ahead;
    ahead.b = first_request;
    ahead.span = span_of(a, ahead.b);
    ahead.tiles = tiles_of<Cfg::TILE>(ahead.span);
    ahead.head = static_cast<int>((x0 - first_before) / ahead.tiles);
    ahead.t = static_cast<uint32_t>((x0 - first_before) % ahead.tiles);
    Cursor now = ahead;
    const bool first_is_cut = now.t > 0;  // the first head's tiles before these belong to an earlier CTA

    // ---- copies: a lane finds a key's row, the warp copies KEYS of them
    const uint32_t ring = frag::smem_addr(smem) + warp * (STAGES * Cfg::STEP_BYTES);
    const uint32_t page_size = a.cache.page_size;
    const bool pow2 = (page_size & (page_size - 1)) == 0;
    const int page_shift = __ffs(page_size) - 1;
    const auto token_of = [&]() { return ahead.span.begin + ahead.t * Cfg::TILE + warp * KEYS + (lane & (KEYS - 1)); };
    const auto page_of = [&]() -> int {  // the page id of this lane's key, a step before it is needed
        const uint32_t token = token_of();
        if (ahead.b >= a.requests || token >= ahead.span.end) return 0;
        const uint32_t index = pow2 ? token >> page_shift : token / page_size;
        return index < static_cast<uint32_t>(a.table_width) ? __ldg(a.table + ahead.b * a.table_stride + index) : -1;
    };
    const auto issue = [&](int stage, int page) {
        const uint32_t token = token_of();
        const uint32_t in_page = pow2 ? token & (page_size - 1) : token % page_size;
        const int kv = ahead.head / heads.groups;
        // (-1: behind the length, zeros; -2: no such page, NaN)
        long long k_at = -1, v_at = -1;
        if (token < ahead.span.end) {
            const bool known = page >= 0 && page < a.cache.pages;
            k_at = known ? (page * a.cache.k_stride[0] + in_page * a.cache.k_stride[1] + kv * a.cache.k_stride[2]) * static_cast<int>(sizeof(C)) : -2;
            v_at = known ? (page * a.cache.v_stride[0] + in_page * a.cache.v_stride[1] + kv * a.cache.v_stride[2]) * static_cast<int>(sizeof(C)) : -2;
        }
        constexpr int CHUNKS = ROW_BYTES / 16, PER_PASS = 32 / CHUNKS;
        const uint32_t to = ring + stage * Cfg::STEP_BYTES;
        const int chunk = lane % CHUNKS;
#pragma unroll
        for (int p = 0; p < KEYS / PER_PASS; ++p) {
            const int row = p * PER_PASS + lane / CHUNKS;
            const long long k_row = __shfl_sync(0xffffffffu, k_at, row), v_row = __shfl_sync(0xffffffffu, v_at, row);
            const uint32_t k_to = to + place<ROW_BYTES>(row, chunk), v_to = k_to + KEYS * ROW_BYTES;
            if (k_row >= 0) {
                copy16<ROW_BYTES>(k_to, static_cast<const char*>(a.cache.k) + k_row + chunk * 16);
                copy16<ROW_BYTES>(v_to, static_cast<const char*>(a.cache.v) + v_row + chunk * 16);
            } else {
                fill16(k_to, k_row == -1 ? 0u : Cfg::CODES ? 0x7f7f7f7fu : 0x7fff7fffu);
                fill16(v_to, 0u);
            }
        }
    };

    const long long steps = x1 - x0;
    int page = page_of();
    long long issued = 0;
    const auto feed = [&](int stage) {
        if (issued < steps) {
            issue(stage, page);
            advance<Cfg>(ahead, a, heads.cut);
            page = issued + 1 < steps ? page_of() : 0;
        }
        ++issued;
        frag::cp_async_commit();
    };
    for (int s = 0; s < STAGES - 1; ++s) feed(s);

    uint32_t q[MT][DIM / 16][4];
    float factor[MT][2];  // of a row's products: into score log2(e)
    float top[MT][2], total[MT][2], o[MT][DT][4];
    const float scale = a.scale * LOG2E * (Cfg::CODES ? a.cache.k_scale : 1.f);
    const auto begin_head = [&]() {
        const int kv = now.head / heads.groups, row0 = (now.head % heads.groups) * Cfg::ROWS;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int row = row0 + m * 16 + half * 8 + g;
                const T* from = static_cast<const T*>(a.q) + now.b * a.q_stride[0] + (static_cast<long long>(kv) * heads.group + row) * a.q_stride[1];
                const bool real = row < heads.group;
                factor[m][half] = scale;
                top[m][half] = -INFINITY, total[m][half] = 0.f;
                if (!Cfg::CODES) {
#pragma unroll
                    for (int d = 0; d < DIM / 16; ++d) {
                        q[m][d][half] = real ? *reinterpret_cast<const uint32_t*>(from + d * 16 + quad * 2) : 0u;
                        q[m][d][half + 2] = real ? *reinterpret_cast<const uint32_t*>(from + d * 16 + 8 + quad * 2) : 0u;
                    }
                } else {
                    // an e4m3 row's dims 4 quad .. 4 quad + 3 come in one word, so the query's dims are dealt the same way. The
                    // product is of f16: a bf16 query's row is first scaled by a power of two to 1 <= max < 2, so that it fits
                    // (what falls below 2^-24 of the row's maximum is rounded away, far below the query's own 2^-8 steps)
                    uint2 raw[DIM / 16];
                    float most = 0.f;
#pragma unroll
                    for (int d = 0; d < DIM / 16; ++d) {
                        raw[d] = real ? *reinterpret_cast<const uint2*>(from + d * 16 + quad * 4) : make_uint2(0u, 0u);
                        const T* x = reinterpret_cast<const T*>(&raw[d]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(to_f32(x[e])));
                    }
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    int power = ((__float_as_int(most) >> 23) & 255) - 127;
                    power = std::is_same<T, __half>::value ? 0 : max(-100, min(power, 120));
                    const float down = __int_as_float((127 - power) << 23);
                    factor[m][half] = scale * __int_as_float((127 + power) << 23);
#pragma unroll
                    for (int d = 0; d < DIM / 16; ++d) {
                        const T* x = reinterpret_cast<const T*>(&raw[d]);
                        q[m][d][half] = frag::pack_f32<false>(to_f32(x[0]) * down, to_f32(x[1]) * down);
                        q[m][d][half + 2] = frag::pack_f32<false>(to_f32(x[2]) * down, to_f32(x[3]) * down);
                    }
                }
            }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[m][d][e] = 0.f;
    };

    float* const merge = reinterpret_cast<float*>(smem + WARPS * STAGES * Cfg::STEP_BYTES);
    // the warps' maxima, sums and outputs of a head become one, eight rows at a time; whole heads go out, cut ones to a piece
    const auto end_head = [&](float* piece) {
        const int kv = now.head / heads.groups, row0 = (now.head % heads.groups) * Cfg::ROWS;
        const int rows = min(Cfg::ROWS, heads.group - row0);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int base = m * 16 + half * 8;
                if (base >= rows) break;
                float sum = total[m][half];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                __syncthreads();  // the last eight rows are read
                if (base + g < rows) {
                    float* to = merge + (warp * 8 + g) * Cfg::PITCH;
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        if (Cfg::CODES) {  // tiles 2d and 2d + 1 hold the even and odd dims of 16
                            if (d % 2 == 0)
                                *reinterpret_cast<float4*>(to + d * 8 + quad * 4) = make_float4(o[m][d][half * 2], o[m][d + 1 < DT ? d + 1 : d][half * 2], o[m][d][half * 2 + 1], o[m][d + 1 < DT ? d + 1 : d][half * 2 + 1]);
                        } else {
                            *reinterpret_cast<float2*>(to + d * 8 + quad * 2) = make_float2(o[m][d][half * 2], o[m][d][half * 2 + 1]);
                        }
                    }
                    if (quad == 0) to[DIM] = top[m][half], to[DIM + 1] = sum;
                }
                __syncthreads();
                for (int i = tid; i < 8 * (DIM / 4); i += THREADS) {
                    const int r = i / (DIM / 4), d = i % (DIM / 4) * 4;
                    if (base + r >= rows) break;
                    float best = -INFINITY;
#pragma unroll
                    for (int w = 0; w < WARPS; ++w) best = fmaxf(best, merge[(w * 8 + r) * Cfg::PITCH + DIM]);
                    const float ref = best == -INFINITY ? 0.f : best;
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                    float s = 0.f;
#pragma unroll
                    for (int w = 0; w < WARPS; ++w) {
                        const float* from = merge + (w * 8 + r) * Cfg::PITCH;
                        const float f = exp2_(from[DIM] - ref);
                        const float4 x = *reinterpret_cast<const float4*>(from + d);
                        acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
                        s += f * from[DIM + 1];
                    }
                    if (piece) {
                        float* to = piece + (base + r) * Cfg::PITCH;
                        *reinterpret_cast<float4*>(to + d) = acc;
                        if (d == 0) to[DIM] = best, to[DIM + 1] = s;
                    } else {
                        const float inv = s == 0.f ? 0.f : (Cfg::CODES ? a.cache.v_scale : 1.f) / s;
                        const long long h = static_cast<long long>(kv) * heads.group + row0 + base + r;
                        uint2 packed;
                        packed.x = frag::pack_f32<std::is_same<T, __nv_bfloat16>::value>(acc.x * inv, acc.y * inv);
                        packed.y = frag::pack_f32<std::is_same<T, __nv_bfloat16>::value>(acc.z * inv, acc.w * inv);
                        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + now.b * a.out_stride[0] + h * a.out_stride[1] + d) = packed;
                        if (a.lse && d == 0) a.lse[now.b * static_cast<long long>(a.heads) + h] = s == 0.f ? -INFINITY : best * LN2 + logf(s);
                    }
                }
            }
    };

    begin_head();
    int stage = 0;
    bool cut_in_front = first_is_cut;
    Record record{0, 0, 0, 0};
    for (long long step = 0; step < steps; ++step) {
        frag::cp_async_wait<STAGES - 2>();
        __syncwarp();
        feed(stage == 0 ? STAGES - 1 : stage - 1);
        const uint32_t from = ring + stage * Cfg::STEP_BYTES;
        stage = stage + 1 == STAGES ? 0 : stage + 1;

        // ---- scores
        float s[MT][NT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[m][j][e] = 0.f;
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) {
            const int row = j * 16 + (lane & 7) + ((lane & 16) >> 1), chunk = (lane >> 3) & 1;
            if (!Cfg::CODES) {
#pragma unroll
                for (int d = 0; d < DIM / 16; ++d) {
                    uint32_t r[4];
                    load4(r, from + place<ROW_BYTES>(row, d * 2 + chunk));
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        frag::mma_f32<Cfg::BF16>(s[m][2 * j], q[m][d], reinterpret_cast<const uint32_t(&)[2]>(r[0]));
                        frag::mma_f32<Cfg::BF16>(s[m][2 * j + 1], q[m][d], reinterpret_cast<const uint32_t(&)[2]>(r[2]));
                    }
                }
            } else {
#pragma unroll
                for (int d = 0; d < DIM / 16; d += 2) {
                    uint32_t r[4];
                    load4(r, from + place<ROW_BYTES>(row, d + chunk));
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint32_t w[2];
                        widen4(r[i], w[0], w[1]);
#pragma unroll
                        for (int m = 0; m < MT; ++m) frag::mma_f32<false>(s[m][2 * j + i / 2], q[m][d + i % 2], w);
                    }
                }
            }
        }

        // ---- softmax
        const uint32_t token0 = now.span.begin + now.t * Cfg::TILE + warp * KEYS;
        const bool ragged = token0 + KEYS > now.span.end;
        uint32_t p[MT][NT / 2][4];
        bool moved = false;
        float keep[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float most = top[m][half];
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = s[m][j][half * 2 + e];
                        x *= factor[m][half];
                        if (ragged && token0 + j * 8 + quad * 2 + e >= now.span.end) x = -INFINITY;
                        most = fmaxf(most, x);
                    }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const float ref = most == -INFINITY ? 0.f : most;
                keep[m][half] = exp2_(top[m][half] - ref);
                moved |= top[m][half] != most;
                top[m][half] = most;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const float u = exp2_(s[m][j][half * 2] - ref), v = exp2_(s[m][j][half * 2 + 1] - ref);
                    sum += u + v;
                    // the weights' one rounding: the product with the values takes 16-bit operands (f16 or bf16)
                    p[m][j / 2][half + (j % 2) * 2] = frag::pack_f32<Cfg::BF16>(u, v);
                }
                total[m][half] = total[m][half] * keep[m][half] + sum;
            }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[m][d][e] *= keep[m][e / 2];
        }

        // ---- values
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) {
            const int row = j * 16 + (lane & 15), chunk = lane >> 4;
            const uint32_t values = from + KEYS * ROW_BYTES;
            if (!Cfg::CODES) {
#pragma unroll
                for (int d = 0; d < DT; d += 2) {
                    uint32_t r[4];
                    load4_trans(r, values + place<ROW_BYTES>(row, d + chunk));
#pragma unroll
                    for (int m = 0; m < MT; ++m) {
                        frag::mma_f32<Cfg::BF16>(o[m][d], p[m][j], reinterpret_cast<const uint32_t(&)[2]>(r[0]));
                        frag::mma_f32<Cfg::BF16>(o[m][d + 1], p[m][j], reinterpret_cast<const uint32_t(&)[2]>(r[2]));
                    }
                }
            } else {
#pragma unroll
                for (int d = 0; d < DT; d += 4) {  // 32 dims: two chunks of a row
                    uint32_t r[4];
                    load4_trans(r, values + place<ROW_BYTES>(row, d / 2 + chunk));
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        // a word holds dims (2g, 2g + 1) of two keys: sorted by dim, the even dims make one tile and the odd another
                        uint32_t even[2], odd[2];
                        widen4(__byte_perm(r[2 * c], 0, 0x3120), even[0], odd[0]);
                        widen4(__byte_perm(r[2 * c + 1], 0, 0x3120), even[1], odd[1]);
#pragma unroll
                        for (int m = 0; m < MT; ++m) {
                            frag::mma_f32<false>(o[m][d + 2 * c], p[m][j], even);
                            frag::mma_f32<false>(o[m][d + 2 * c + 1], p[m][j], odd);
                        }
                    }
                }
            }
        }

        // ---- the end of a head, or of the share
        const bool head_ends = now.t + 1 == now.tiles, share_ends = step + 1 == steps;
        if (head_ends || share_ends) {
            float* piece = nullptr;
            if (cut_in_front || !head_ends) piece = pieces + (2ll * blockIdx.x + (cut_in_front ? 0 : 1)) * (Cfg::ROWS * Cfg::PITCH);
            end_head(piece);
            if (!head_ends && !cut_in_front) {  // the head starts here and goes on: the CTAs up to the one that holds its last tile
                const long long last = x1 - 1 + (now.tiles - 1 - now.t);
                record = {now.b, now.head, static_cast<int>(((last + 1) * n + all - 1) / all - 1 - blockIdx.x + 1), 0};
            }
            cut_in_front = false;
        }
        advance<Cfg>(now, a, heads.cut);
        if (head_ends && !share_ends) begin_head();
    }
    if (tid == 0) records[blockIdx.x] = record;
}

// The pieces of the heads that were cut: CTA c adds up those of the head that starts in CTA c's share and goes on. A row's
// maximum and sum are joined as in the kernel above, always in the keys' order, so results do not depend on timing.
template <class T, class C, int DIM, int MT>
__global__ void __launch_bounds__(128) paged_join_kernel(const emb_paged_attend_t a, const Record* records, const float* pieces) {
    using Cfg = Config<T, C, DIM, MT>;
    follow_on();
    const Record record = records[blockIdx.x];
    if (record.pieces == 0) return;
    const Heads heads(a, Cfg::ROWS);
    const int kv = record.head / heads.groups, row0 = (record.head % heads.groups) * Cfg::ROWS;
    const int rows = min(Cfg::ROWS, heads.group - row0);
    const auto piece_of = [&](int i, int row) {
        return pieces + (2ll * (blockIdx.x + i) + (i == 0)) * (Cfg::ROWS * Cfg::PITCH) + row * Cfg::PITCH;
    };
    for (int i = threadIdx.x; i < rows * (DIM / 4); i += blockDim.x) {
        const int r = i / (DIM / 4), d = i % (DIM / 4) * 4;
        float best = -INFINITY;
        for (int k = 0; k < record.pieces; ++k) best = fmaxf(best, piece_of(k, r)[DIM]);
        const float ref = best == -INFINITY ? 0.f : best;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float s = 0.f;
#pragma unroll 4
        for (int k = 0; k < record.pieces; ++k) {
            const float* from = piece_of(k, r);
            const float f = exp2_(from[DIM] - ref);
            const float4 x = *reinterpret_cast<const float4*>(from + d);
            acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
            s += f * from[DIM + 1];
        }
        const float inv = s == 0.f ? 0.f : (Cfg::CODES ? a.cache.v_scale : 1.f) / s;
        const long long h = static_cast<long long>(kv) * heads.group + row0 + r;
        uint2 packed;
        packed.x = frag::pack_f32<std::is_same<T, __nv_bfloat16>::value>(acc.x * inv, acc.y * inv);
        packed.y = frag::pack_f32<std::is_same<T, __nv_bfloat16>::value>(acc.z * inv, acc.w * inv);
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + record.request * a.out_stride[0] + h * a.out_stride[1] + d) = packed;
        if (a.lse && d == 0) a.lse[record.request * static_cast<long long>(a.heads) + h] = s == 0.f ? -INFINITY : best * LN2 + logf(s);
    }
}

constexpr int MAX_DEVICES = 64;

// SMs of the current device; 0 and an error text where that cannot be had
int sm_count() {
    static int known[MAX_DEVICES];  // (threads that race here store the same number)
    int device = -1;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= MAX_DEVICES) return 0;
    if (!known[device]) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
        known[device] = n;
    }
    return known[device];
}

template <class Cfg> int64_t piece_bytes() { return 2ll * Cfg::ROWS * Cfg::PITCH * 4; }

// the CTAs of a launch: as many as the SMs hold at once
template <class Cfg> int grid_of(const emb_paged_attend_t& a, int sms) {
    const int64_t longest = a.window ? min(static_cast<int64_t>(a.window), static_cast<int64_t>(a.table_width) * a.cache.page_size + 1) : static_cast<int64_t>(a.table_width) * a.cache.page_size + 1;
    const double most = static_cast<double>(a.requests) * Heads(a, Cfg::ROWS).cut * ((longest + Cfg::TILE - 1) / Cfg::TILE);
    const int all = sms * Cfg::CTAS;
    return most < all ? static_cast<int>(most) : all;
}

template <class T, class C, int DIM, int MT> int run(const emb_paged_attend_t& a, cudaStream_t stream, int64_t* need) {
    using Cfg = Config<T, C, DIM, MT>;
    const int sms = sm_count();
    if (!sms) return refuse("paged_attend: the current device cannot be asked for its SMs");
    const int grid = grid_of<Cfg>(a, sms);
    const int64_t bytes = grid * (static_cast<int64_t>(sizeof(Record)) + piece_bytes<Cfg>());
    if (need) {
        *need = bytes;
        return 0;
    }
    if (a.workspace_bytes < bytes || !a.workspace || !aligned16(a.workspace))
        return refuse("paged_attend: a workspace of %lld bytes (16-byte aligned) is needed, not %lld", static_cast<long long>(bytes), static_cast<long long>(a.workspace_bytes));
    auto kernel = paged_attend_kernel<T, C, DIM, MT>;
    static std::once_flag once[MAX_DEVICES];
    int device = 0;
    cudaGetDevice(&device);
    std::call_once(once[device], [&] { cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM); });
    Record* records = static_cast<Record*>(a.workspace);
    float* pieces = reinterpret_cast<float*>(records + grid);
    if (int r = launched("launch of paged_attend", launch(kernel, grid, THREADS, Cfg::SMEM, stream, a, records, pieces))) return r;
    return launched("launch of paged_join", launch(paged_join_kernel<T, C, DIM, MT>, grid, 128, 0, stream, a, records, pieces));
}

template <class T, class C> int run_dim(const emb_paged_attend_t& a, cudaStream_t stream, int64_t* need) {
    const bool wide = a.heads / a.cache.kv_heads > 16;
    switch (a.cache.dim) {
        case 64: return wide ? run<T, C, 64, 2>(a, stream, need) : run<T, C, 64, 1>(a, stream, need);
        case 128: return wide ? run<T, C, 128, 2>(a, stream, need) : run<T, C, 128, 1>(a, stream, need);
        default: return run<T, C, 256, 1>(a, stream, need);
    }
}

int attend(const emb_paged_attend_t* args, void* stream, int64_t* need) {
    if (!args) return refuse("paged_attend: null arguments");
    const emb_paged_attend_t& a = *args;
    if (int r = check_cache("paged_attend", a.cache, a.dtype)) return r;
    if (a.requests < 0 || a.heads < 1 || a.heads > 65535 || a.heads % a.cache.kv_heads)
        return refuse("paged_attend: %d requests of %d heads over %d key heads: a multiple of the key heads", a.requests, a.heads, a.cache.kv_heads);
    if (a.table_width < 1 || static_cast<int64_t>(a.table_width) * a.cache.page_size >= (1ll << 31) || a.table_stride < 0)
        return refuse("paged_attend: a table row of %d pages of %d tokens", a.table_width, a.cache.page_size);
    if (a.window < 0) return refuse("paged_attend: a negative window");
    if (!(a.scale > -INFINITY && a.scale < INFINITY)) return refuse("paged_attend: the scale is not a finite number");
    if (need) *need = 0;
    if (a.requests == 0) return 0;
    if (!need) {
        if (!a.table || !a.lengths) return refuse("paged_attend: null table or lengths");
        if (!a.q || !a.out || !aligned16(a.q) || !aligned16(a.out)) return refuse("paged_attend: q or out is null or not 16-byte aligned");
        for (const int64_t* s : {a.q_stride, a.out_stride})
            if (!stride_fits(s[0], 2) || !stride_fits(s[1], 2)) return refuse("paged_attend: a stride of q or out is not a multiple of 16 bytes below 2^32 elements");
        const int64_t rows[2] = {a.requests, a.heads};
        if (!rows_apart(rows, a.out_stride, a.cache.dim)) return refuse("paged_attend: rows of out overlap");
    }
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.dtype == EMB_F16) return a.cache.dtype == EMB_U8 ? run_dim<__half, E4m3>(a, s, need) : run_dim<__half, __half>(a, s, need);
    return a.cache.dtype == EMB_U8 ? run_dim<__nv_bfloat16, E4m3>(a, s, need) : run_dim<__nv_bfloat16, __nv_bfloat16>(a, s, need);
}

}  // namespace

extern "C" int emb_paged_attend(const emb_paged_attend_t* args, void* stream) { return attend(args, stream, nullptr); }

extern "C" int64_t emb_paged_attend_workspace(const emb_paged_attend_t* args) {
    int64_t need = 0;
    const int r = attend(args, nullptr, &need);
    return r ? (r < 0 ? r : -static_cast<int64_t>(r)) : need;
}
