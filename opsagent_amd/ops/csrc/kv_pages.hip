// Copies of cache pages, in the tensors of all layers at once, for MI355X (gfx950).
//
// A sequence that forks copies the page it is about to write into, as far as that is filled; a
// cache that is compacted moves whole pages. Each copy is `tokens` rows of `row` bytes from the
// start of page src to that of page dst, the same in every tensor. What bounds it is memory
// alone: read once, written once.
//
// Tables of bases and copies go with the launch, by value: nothing has to outlive the call, and a
// captured launch keeps its own. Up to 192 tensors (the 160 of an 80-layer model) and 192 copies
// fit in the 4 KiB that a launch may carry; more take more launches.

#include "common.h"

constexpr int MAX_TENSORS = 192, MAX_COPIES = 192;

struct PageTensors {
    char* base[MAX_TENSORS];
};
struct PageCopies {
    int src[MAX_COPIES], dst[MAX_COPIES], tokens[MAX_COPIES];
};
static_assert(sizeof(PageTensors) + sizeof(PageCopies) + 32 <= 4096, "what a launch may carry");

// Grid: slices of a page, tensors, copies. A thread has UNROLL pieces of 16 bytes in flight.
constexpr int UNROLL = 4;
__global__ __launch_bounds__(256) void kv_pages_copy_kernel(PageTensors tensors, PageCopies copies,
                                                            int64_t step, int row) {
    char* const base = tensors.base[blockIdx.y];
    const int c = blockIdx.z;
    const int64_t bytes = (int64_t)copies.tokens[c] * row;
    const char* src = base + copies.src[c] * step;
    char* dst = base + copies.dst[c] * step;
    const int64_t at = ((int64_t)blockIdx.x * UNROLL * 256 + threadIdx.x) * 16;
    uint4 part[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i)
        if (at + i * 4096 < bytes) part[i] = *reinterpret_cast<const uint4*>(src + at + i * 4096);
#pragma unroll
    for (int i = 0; i < UNROLL; ++i)
        if (at + i * 4096 < bytes) *reinterpret_cast<uint4*>(dst + at + i * 4096) = part[i];
}

// bases: `tensors` addresses on the host, each of `pages` pages `step` bytes apart, a page `block`
// rows of `row` bytes. copies: src, dst and tokens of each copy, on the host.
extern "C" int oa_kv_pages_copy(void* stream, const uint64_t* bases, int tensors, int64_t step, int row,
                                int block, int pages, const int* copies, int n) {
    if (tensors < 0 || n < 0 || row < 16 || row % 16 != 0 || step % 16 != 0 || block < 1 || pages < 1)
        return -100;
    if ((int64_t)block * row > INT32_MAX) return -101;
    for (int i = 0; i < tensors; ++i)
        if (bases[i] % 16 != 0) return -103;
    for (int i = 0; i < n; ++i) {
        const int* c = copies + 3 * i;
        if (c[0] < 0 || c[0] >= pages || c[1] < 0 || c[1] >= pages || c[2] < 0 || c[2] > block) return -104;
    }
    for (int t0 = 0; t0 < tensors; t0 += MAX_TENSORS) {
        const int nt = min(MAX_TENSORS, tensors - t0);
        PageTensors t;
        for (int i = 0; i < nt; ++i) t.base[i] = reinterpret_cast<char*>(bases[t0 + i]);
        for (int c0 = 0; c0 < n; c0 += MAX_COPIES) {
            const int nc = min(MAX_COPIES, n - c0);
            PageCopies c;
            int most = 0;
            for (int i = 0; i < nc; ++i) {
                const int* p = copies + 3 * (c0 + i);
                c.src[i] = p[0];
                c.dst[i] = p[1];
                c.tokens[i] = p[2];
                most = max(most, p[2]);
            }
            if (!most) continue;
            const int64_t slices = CEIL_DIV((int64_t)most * row, UNROLL * 4096);
            hipLaunchKernelGGL(kv_pages_copy_kernel, dim3((unsigned)slices, nt, nc), dim3(256), 0,
                               (hipStream_t)stream, t, c, step, row);
            HIP_CHECK_LAUNCH();
        }
    }
    return 0;
}
