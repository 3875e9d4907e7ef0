// emb_paged_assign: page tables and slot maps of a serving step, from the requests' lengths, on the GPU.
//
// Two prefix sums over the requests (new rows, new pages) decide everything; no request's pages depend on a value that
// another thread writes, so one launch does it: every CTA sums over all requests (lengths are a few KB and stay in L2) and
// takes ROWS rows of the step. A request that has rows there leaves what they need to know at the place of its first one; a
// running maximum over the places then gives each row its request. A page that is new to a request is entered into the
// table by the row that is its first token: the page of a row behind it comes from the free list, not from the table, so
// rows never wait for one another. Sums saturate at 2^31 - 1, beyond anything that can be granted.
// Bound by latency (a launch, loads of lengths, a scan, loads of pages): the traffic is 8 bytes a row. (One request a
// thread, a scan for each sum and a bisection for each row took 12.2 us with a cold L2 for 1000 requests with up to 512
// new tokens, where this takes 6.2; a kernel that does nothing takes 2.2 so measured.)

#include "paged_common.cuh"

namespace {

using namespace emb::paged;

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int ITEMS = 4;            // requests of a thread per pass
constexpr int ROWS = 2 * THREADS;   // rows of the step per CTA
constexpr uint32_t MOST = 0x7fffffffu;

struct Request {  // of a row
    int32_t start, id, cached, have;
    int32_t first, granted;  // its first new page's place in the free list
};

__device__ __forceinline__ uint32_t sum_of(uint32_t a, uint32_t b) { return min(a + b, MOST); }

__global__ void __launch_bounds__(THREADS) paged_assign_kernel(const emb_paged_assign_t a, const Divisor page_size) {
    __shared__ Request at[ROWS];
    __shared__ int place[ROWS];  // of the request that starts at a row (or goes on at row 0): the row + 1; else 0
    __shared__ uint32_t row_slab[WARPS], page_slab[WARPS];
    __shared__ int top_slab[WARPS];
    __shared__ unsigned taken_all, refused_all;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int i = tid; i < ROWS; i += THREADS) place[i] = 0;
    if (tid == 0) taken_all = refused_all = 0;
    follow_on();
    const uint32_t row0 = blockIdx.x * ROWS, tokens = a.tokens, row1 = min(row0 + ROWS, tokens);
    const uint32_t head = min(max(*a.free_head, 0), a.free_count), room = a.free_count - head;
    const uint32_t capacity = static_cast<uint32_t>(a.table_width) * page_size.d;
    const auto pages_for = [&](uint32_t n) { return n ? page_size.over(n - 1) + 1 : 0u; };

    uint32_t rows_done = 0, pages_done = 0, taken = 0, refused = 0;
    for (int base = 0; base < a.requests; base += THREADS * ITEMS) {
        uint32_t cached[ITEMS], fresh[ITEMS], have[ITEMS], need[ITEMS], rows = 0, pages = 0;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int b = base + tid * ITEMS + k;
            cached[k] = b < a.requests ? max(a.cached[b], 0) : 0;
            fresh[k] = b < a.requests ? max(a.fresh[b], 0) : 0;
        }
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            have[k] = pages_for(cached[k]);
            // (a request that does not fit its table row asks for nothing; one that does not fit the step's rows stands behind all
            // that do, so what it asks for changes nothing)
            need[k] = fresh[k] && cached[k] + fresh[k] <= capacity ? pages_for(cached[k] + fresh[k]) - have[k] : 0u;
            rows = sum_of(rows, fresh[k]), pages = sum_of(pages, need[k]);
        }
        uint32_t rows_upto = rows, pages_upto = pages;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t r = __shfl_up_sync(0xffffffffu, rows_upto, d), p = __shfl_up_sync(0xffffffffu, pages_upto, d);
            if (lane >= d) rows_upto = sum_of(rows_upto, r), pages_upto = sum_of(pages_upto, p);
        }
        // (what stands before this thread's requests; a saturated sum stays saturated: it is not taken back by a subtraction)
        uint32_t row_before = __shfl_up_sync(0xffffffffu, rows_upto, 1), page_before = __shfl_up_sync(0xffffffffu, pages_upto, 1);
        if (lane == 0) row_before = page_before = 0;
        __syncthreads();  // the slabs' last readers are done, and `place` is cleared
        if (lane == 31) row_slab[warp] = rows_upto, page_slab[warp] = pages_upto;
        __syncthreads();
        uint32_t start = rows_done, upto = pages_done;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) start = sum_of(start, row_slab[w]), upto = sum_of(upto, page_slab[w]);
            rows_done = sum_of(rows_done, row_slab[w]), pages_done = sum_of(pages_done, page_slab[w]);
        }
        start = sum_of(start, row_before), upto = sum_of(upto, page_before);
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int b = base + tid * ITEMS + k;
            const uint32_t end = sum_of(start, fresh[k]), first = upto;
            upto = sum_of(upto, need[k]);
            // the needs' running sum only grows, so the requests that get pages are those before the first one that does not
            const bool granted = !fresh[k] || (cached[k] + fresh[k] <= capacity && end <= tokens && (!need[k] || upto <= room));
            refused += !granted;
            if (granted && need[k]) taken = upto;
            if (fresh[k] && start < row1 && end > row0) {
                const uint32_t row = max(start, row0) - row0;
                place[row] = row + 1;
                at[row] = {static_cast<int32_t>(start), b, static_cast<int32_t>(cached[k]), static_cast<int32_t>(have[k]), static_cast<int32_t>(head + first), granted};
            }
            if (blockIdx.x == 0 && b < a.requests) {
                a.starts[b] = start;
                a.lengths[b] = granted ? cached[k] + fresh[k] : cached[k];
            }
            start = end;
        }
    }
    __syncthreads();  // `place` and `at` are whole

    // the last place at or before each row; a thread has two rows side by side
    const int p0 = place[tid * 2], p1 = max(p0, place[tid * 2 + 1]);
    int upto = p1;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto = max(upto, x);
    }
    int before = __shfl_up_sync(0xffffffffu, upto, 1);
    if (lane == 0) before = 0;
    if (lane == 31) top_slab[warp] = upto;
    if (blockIdx.x == 0) {
        if (refused) atomicAdd(&refused_all, refused);
        if (taken) atomicMax(&taken_all, taken);
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
        if (w < warp) before = max(before, top_slab[w]);
    if (blockIdx.x == 0 && tid == 0) {
        a.starts[a.requests] = rows_done;
        *a.free_head_out = head + taken_all;
        a.report[0] = taken_all;
        a.report[1] = refused_all;
        a.report[2] = rows_done > tokens ? rows_done - tokens : 0;
        a.report[3] = rows_done;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const uint32_t i = row0 + tid * 2 + u;
        if (i >= row1) break;
        const int from = max(before, u ? p1 : p0);
        int32_t slot = -1, position = 0;
        if (i < rows_done && from) {
            const Request r = at[from - 1];
            const uint32_t pos = sum_of(r.cached, i - r.start);
            position = pos;
            if (r.granted) {
                const uint32_t index = page_size.over(pos), in_page = pos - index * page_size.d;
                int32_t* const entry = a.table + r.id * a.table_stride + index;
                int32_t page;
                if (index < static_cast<uint32_t>(r.have)) {
                    page = *entry;
                } else {
                    page = a.free_pages[r.first + (index - r.have)];
                    if (in_page == 0) *entry = page;
                }
                const long long s = static_cast<long long>(page) * page_size.d + in_page;
                if (page >= 0 && s <= MOST) slot = static_cast<int32_t>(s);
            }
        }
        a.slots[i] = slot;
        a.positions[i] = position;
    }
}

}  // namespace

extern "C" int emb_paged_assign(const emb_paged_assign_t* args, void* stream) {
    if (!args) return refuse("paged_assign: null arguments");
    const emb_paged_assign_t& a = *args;
    if (static_cast<int64_t>(a.table_width) * a.page_size >= (1ll << 31)) return refuse("paged_assign: a table row of 2^31 tokens or more");
    if (a.tokens > (1ll << 31) - 1024) return refuse("paged_assign: 2^31 rows or more");
    if (a.requests < 0 || a.table_width < 1 || a.free_count < 0 || a.page_size < 1 || a.tokens < 0 || a.table_stride < 0)
        return refuse("paged_assign: a count is negative, or the table width or page size below 1");
    if ((a.requests && (!a.cached || !a.fresh || !a.table || !a.lengths)) || (a.free_count && !a.free_pages) ||
        (a.tokens && (!a.slots || !a.positions)) || !a.free_head || !a.starts || !a.free_head_out || !a.report)
        return refuse("paged_assign: null pointer");
    if (a.requests > 1 && a.table_stride < a.table_width) return refuse("paged_assign: rows of the table overlap");
    if (a.lengths && (a.lengths == a.cached || a.lengths == a.fresh)) return refuse("paged_assign: lengths may not be cached or fresh");
    if (a.free_head_out == a.free_head) return refuse("paged_assign: free_head_out may not be free_head");
    const auto ints = [](const char* name, const void* p, int64_t n) { return Area(name, p, n * 4); };
    const int64_t requests = a.requests;
    const Area written[7] = {ints("table", a.table, requests ? a.table_width : 0).by(requests, a.table_stride * 4), ints("slots", a.slots, a.tokens), ints("positions", a.positions, a.tokens),
                             ints("starts", a.starts, requests + 1), ints("lengths", a.lengths, requests), ints("free_head_out", a.free_head_out, 1), ints("report", a.report, 4)};
    const Area read[4] = {ints("cached", a.cached, requests), ints("fresh", a.fresh, requests), ints("free_pages", a.free_pages, a.free_count), ints("free_head", a.free_head, 1)};
    const char* which[2];
    if (touches(written, read, nullptr, which)) return refuse("paged_assign: %s and %s share memory", which[0], which[1]);
    const unsigned grid = a.tokens > ROWS ? (static_cast<unsigned>(a.tokens) + ROWS - 1) / ROWS : 1u;
    return launched("launch of paged_assign", launch(paged_assign_kernel, dim3(grid), THREADS, 0, static_cast<cudaStream_t>(stream), a, Divisor(a.page_size)));
}
