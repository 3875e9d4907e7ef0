// emb_paged_assign: page tables and slot maps of a serving step, from the requests' lengths, on the GPU.
//
// Two prefix sums over the requests (new rows, new pages) decide everything; no request's pages depend on a value that
// another thread writes, so one launch does it: every CTA sums over all requests (lengths are a few KB and stay in L2)
// and keeps the requests whose rows meet its own ROWS rows of the step; then a thread per row finds its request among
// them by bisection. A page that is new to a request is entered into the table by the row that is its first token: the
// page of a row behind it comes from the free list, not from the table, so rows never wait for one another.
// Bound by latency (one launch, two dependent loads and a scan): the traffic is 8 bytes a row.

#include "paged_common.cuh"

namespace {

using namespace emb::paged;

constexpr int THREADS = 256;
constexpr int ROWS = 1024;  // rows of the step per CTA

struct Meets {  // a request whose rows meet this CTA's
    int32_t start, request, cached, have;
    long long first;  // of its new pages in the free list; -1: refused
};

struct Sums {
    long long x;
    int32_t y;
};

__device__ __forceinline__ Sums operator+(const Sums& a, const Sums& b) { return {a.x + b.x, a.y + b.y}; }

// inclusive sums over the CTA's threads in thread order, and over all of them
__device__ __forceinline__ Sums block_scan(Sums v, Sums (&slab)[THREADS / 32], Sums& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, v.x, d);
        const int32_t y = __shfl_up_sync(0xffffffffu, v.y, d);
        if (lane >= d) v.x += x, v.y += y;
    }
    __syncthreads();  // the slab's last readers are done
    if (lane == 31) slab[warp] = v;
    __syncthreads();
    Sums before{0, 0};
    total = {0, 0};
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before = before + slab[w];
        total = total + slab[w];
    }
    return before + v;
}

__device__ __forceinline__ int32_t clamp_i32(long long x) { return x > 0x7fffffffll ? 0x7fffffff : static_cast<int32_t>(x); }

__global__ void __launch_bounds__(THREADS) paged_assign_kernel(const emb_paged_assign_t a) {
    __shared__ Meets meets[ROWS];  // in the requests' order; each of them has a row of this CTA's, so ROWS are enough
    __shared__ Sums slab[THREADS / 32];
    __shared__ long long taken_all;
    __shared__ int refused_all;
    const int tid = threadIdx.x;
    follow_on();
    const long long row0 = static_cast<long long>(blockIdx.x) * ROWS;
    const long long row1 = min(row0 + ROWS, static_cast<long long>(a.tokens));
    const long long head = min(max(*a.free_head, 0), a.free_count), room = a.free_count - head;
    if (tid == 0) taken_all = 0, refused_all = 0;

    long long rows_done = 0, pages_done = 0, taken = 0;
    int met = 0, refused = 0;
    for (int base = 0; base < a.requests; base += THREADS) {
        const int b = base + tid;
        const bool real = b < a.requests;
        const long long c = real ? max(a.cached[b], 0) : 0, f = real ? max(a.fresh[b], 0) : 0;
        const long long have = (c + a.page_size - 1) / a.page_size, want = (c + f + a.page_size - 1) / a.page_size;
        Sums total;
        const long long end = rows_done + block_scan({f, 0}, slab, total).x, start = end - f;
        rows_done += total.x;
        const bool fits = f == 0 || (c + f <= static_cast<long long>(a.table_width) * a.page_size && end <= a.tokens);
        const long long need = fits ? want - have : 0;
        const bool meet = f > 0 && start < row1 && end > row0;
        const Sums upto = Sums{pages_done, met} + block_scan({need, meet}, slab, total);
        pages_done += total.x, met += total.y;
        // the needs' running sum only grows, so the requests that get pages are those before the first one that does not
        const bool granted = fits && (need == 0 || upto.x <= room);
        refused += !granted;
        if (granted && need) taken = upto.x;
        if (meet) meets[upto.y - 1] = {static_cast<int32_t>(start), b, static_cast<int32_t>(c), static_cast<int32_t>(have), granted ? head + upto.x - need : -1};
        if (real && blockIdx.x == 0) {
            a.starts[b] = clamp_i32(start);
            a.lengths[b] = clamp_i32(granted ? c + f : c);
        }
    }
    __syncthreads();  // `meets` is whole
    if (blockIdx.x == 0) {
        if (refused) atomicAdd(&refused_all, refused);
        if (taken) atomicMax(&taken_all, taken);
        __syncthreads();
        if (tid == 0) {
            a.starts[a.requests] = clamp_i32(rows_done);
            *a.free_head_out = static_cast<int32_t>(head + taken_all);
            a.report[0] = static_cast<int32_t>(taken_all);
            a.report[1] = refused_all;
            a.report[2] = clamp_i32(max(rows_done - a.tokens, 0ll));
            a.report[3] = clamp_i32(rows_done);
        }
    }
    for (long long i = row0 + tid; i < row1; i += THREADS) {
        int32_t slot = -1, position = 0;
        if (i < rows_done) {
            int lo = 0, hi = met;  // the last request that starts at or before row i
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (meets[mid].start <= i) lo = mid;
                else hi = mid;
            }
            const Meets m = meets[lo];
            const long long pos = m.cached + (i - m.start);
            position = clamp_i32(pos);
            if (m.first >= 0) {
                const int32_t index = static_cast<int32_t>(pos / a.page_size), in_page = static_cast<int32_t>(pos % a.page_size);
                int32_t* entry = a.table + m.request * a.table_stride + index;
                int32_t page;
                if (index < m.have) {
                    page = *entry;
                } else {
                    page = a.free_pages[m.first + index - m.have];
                    if (in_page == 0) *entry = page;
                }
                const long long s = static_cast<long long>(page) * a.page_size + in_page;
                if (page >= 0 && s <= 0x7fffffffll) slot = static_cast<int32_t>(s);
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
    if (a.requests < 0 || a.table_width < 1 || a.free_count < 0 || a.page_size < 1 || a.tokens < 0 || a.table_stride < 0)
        return refuse("paged_assign: a count is negative, or the table width or page size below 1");
    if ((a.requests && (!a.cached || !a.fresh || !a.table || !a.lengths)) || (a.free_count && !a.free_pages) ||
        (a.tokens && (!a.slots || !a.positions)) || !a.free_head || !a.starts || !a.free_head_out || !a.report)
        return refuse("paged_assign: null pointer");
    if (a.requests > 1 && a.table_stride < a.table_width) return refuse("paged_assign: rows of the table overlap");
    if (a.lengths && (a.lengths == a.cached || a.lengths == a.fresh)) return refuse("paged_assign: lengths may not be cached or fresh");
    if (a.free_head_out == a.free_head) return refuse("paged_assign: free_head_out may not be free_head");
    const unsigned grid = a.tokens > ROWS ? (static_cast<unsigned>(a.tokens) + ROWS - 1) / ROWS : 1u;
    return launched("launch of paged_assign", launch(paged_assign_kernel, grid, THREADS, 0, static_cast<cudaStream_t>(stream), a));
}
