// Copies of cache pages, in the tensors of all layers at once, for MI355X (gfx950).
//
// A sequence that forks copies the page it is about to write into, as far as that is filled; a
// cache that is compacted moves whole pages. Each copy is `tokens` rows of `row` bytes from the
// start of page src to that of page dst, the same in every tensor. What bounds it is memory
// alone: read once, written once.
//
// Tables of bases and copies go with the launch, by value: nothing has to outlive the call, and a
// captured launch keeps its own. Up to 192 tensors (the 160 of an 80-layer model) and 128 copies
// fit in the 4 KiB that a launch may carry; more take more launches. Copies of one source that
// follow each other (a prompt's choices) read it once.

#include "common.h"

constexpr int MAX_TENSORS = 192, MAX_COPIES = 128;

struct PageTensors {
    char* base[MAX_TENSORS];
};
struct PageCopies {                        // source i goes to dst[begin[i]] .. dst[begin[i + 1]]
    int src[MAX_COPIES], tokens[MAX_COPIES], dst[MAX_COPIES];
    uint16_t begin[MAX_COPIES + 1];
};
static_assert(sizeof(PageTensors) + sizeof(PageCopies) + 32 <= 4096, "what a launch may carry");

// Grid: 4-KiB slices of a page, sources, tensors: the copies of a tensor side by side, and 16 bytes a
// thread. What is written is not kept: it is more than the next reader's share of a cache where it
// takes time at all. us, by size: 96 pages of 64 KiB in 64 tensors (805 MB in and out) 128 (6.3 TB/s;
// kept 135, tensors side by side 157, 64 bytes a thread 162), three copies of 16 pages' first tokens in
// 160 tensors (291 MB) 66 (77, 78, 99), three of one in 64 4, with the launch. From one card to another,
// and with how much of the caches the last copy left, those of 16 pages take 47 to 82.
__global__ __launch_bounds__(256) void kv_pages_copy_kernel(PageTensors tensors, PageCopies copies,
                                                            int64_t step, int row) {
    typedef __attribute__((ext_vector_type(4))) uint32_t u4;
    char* const base = tensors.base[blockIdx.z];
    const int c = blockIdx.y;
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 16;
    if (at >= (int64_t)copies.tokens[c] * row) return;
    const u4 piece = *reinterpret_cast<const u4*>(base + copies.src[c] * step + at);
    for (int i = copies.begin[c]; i < copies.begin[c + 1]; ++i)
        __builtin_nontemporal_store(piece, reinterpret_cast<u4*>(base + copies.dst[i] * step + at));
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
            int sources = 0, most = 0;
            for (int i = 0; i < nc; ++i) {
                const int* p = copies + 3 * (c0 + i);
                if (!sources || c.src[sources - 1] != p[0] || c.tokens[sources - 1] != p[2]) {
                    c.src[sources] = p[0];
                    c.tokens[sources] = p[2];
                    c.begin[sources++] = (uint16_t)i;
                }
                c.dst[i] = p[1];
                most = max(most, p[2]);
            }
            c.begin[sources] = (uint16_t)nc;
            if (!most) continue;
            hipLaunchKernelGGL(kv_pages_copy_kernel, dim3((unsigned)CEIL_DIV((int64_t)most * row, 4096), sources, nt),
                               dim3(256), 0, (hipStream_t)stream, t, c, step, row);
            HIP_CHECK_LAUNCH();
        }
    }
    return 0;
}
