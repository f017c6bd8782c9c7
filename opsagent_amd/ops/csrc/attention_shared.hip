// Decode attention of a batch whose sequences begin with the same cache pages, for MI355X (gfx950).
//
// Row b (one new token of a sequence) attends to its n[b] paged keys:
//     out[b, h] = sum_j softmax_j(scale * q[b, h] . k_j) v_j,   zeros where n[b] = 0.
// Row b says that its first shared[b] pages are those of row leaders[b]. Rows with one leader are a
// group, and the pages that all of them share are read once for the group: their (row, head) pairs
// of a key head are the columns of one product with the keys, as many queries of one prompt would
// be. What lies behind is read for each row. Both leave unnormalised sums with the maximum and sum
// of weights that they were taken with, and a second launch adds those up.
//
// Sums, maxima and weight sums are float32. Weights enter the product with the values as 16-bit
// numbers of the cache's type, as the matrix cores take them: off by half a step of each weight, which
// averages out over the keys. Their sum is that of the rounded ones, so that what is divided by is what
// was added up. float16 weights are taken 2^15 times as large, the largest power of 2 below its end:
// those from 2^-29 of the largest on have all their bits, where 2^-14 would be the least. The output is
// rounded to the same type.
//
// What bounds it (us; 32 heads on 8 and 64 on 8 of 128 channels, bfloat16): rows that share nothing, memory
// (48 of up to 2000 tokens, 220 MB, 41: 5.4 TB/s); a few rows, latencies (a block's plan or its record 2
// to 3, first keys 2, a step 1, sums 1; the second launch 3); many rows behind one prefix, matrix and
// vector instructions of steps of 128 columns, 2.2 us for two blocks of a CU and 64 keys (128 rows
// behind 16400 tokens 116 in all, 0.6 PFLOP/s: of 64 blocks of a key head 48 take 44 such steps each, 16 the
// rows' own keys, which end sooner).
//
//   q            [B, Hq, D] 16-bit, rows and heads any multiple of 8 elements apart
//   kc, vc       [pages, 2^shift, Hk, D], pages, tokens and heads any multiple of 8 elements apart
//   block_table  [B, width] int32, rows any number apart
//   plan         ints: see PLAN below, made by shared_plan_kernel from lengths and leaders
//   o_part       [slots, Hq, D] float32, ml_part [slots, Hq, 2]: row b has the slots
//                first[b] .. first[b] + splits[b]

#include "common.h"

typedef __attribute__((ext_vector_type(8))) __bf16 sh_b8;
typedef __attribute__((ext_vector_type(8))) _Float16 sh_h8;
typedef __attribute__((ext_vector_type(4))) short sh_s4;
typedef __attribute__((ext_vector_type(4))) float sh_f4;

template <bool F16>
__device__ __forceinline__ sh_f4 sh_product(uint4 a, uint4 b, sh_f4 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(sh_h8, a), __builtin_bit_cast(sh_h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(sh_b8, a), __builtin_bit_cast(sh_b8, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ uint32_t sh_pack(float lo, float hi) {
    if constexpr (F16) {
        typedef __attribute__((ext_vector_type(2))) _Float16 h2;
        return __builtin_bit_cast(uint32_t, h2{(_Float16)lo, (_Float16)hi});
    } else {
        typedef __attribute__((ext_vector_type(2))) __bf16 b2;
        return __builtin_bit_cast(uint32_t, b2{(__bf16)lo, (__bf16)hi});
    }
}

// ---- plan --------------------------------------------------------------------------------------
// PLAN, in ints: items, sizes of the line (padded to 8) | first[B] | splits[B] | members[B], rows group after group |
// units of 8: table row (-1: none), first key, end, place of the group's tile in members, members of
// the tile (0: the table row alone), split, next unit of the item (-1: none), the table row's first slot.
//
// A block takes items, each a chain of units; item i begins with unit i, and what follows in a chain
// for row b is unit items + b. The items of a key head are to be of one size and as many as it has
// blocks (`runs`). A group's pages are one item for each tile of columns and each of n equal chunks
// of keys, tiles of a chunk side by side, so that they read the same keys at the same time. What lies
// behind is put in a line, row after row, and cut in equal items at multiples of 128 keys of a row.
// Sizes are in 64 keys, and a unit costs UNIT_COST of them beside its keys.
constexpr int PLAN_HEAD = 8, UNIT = 8, UNIT_COST = 1;
constexpr int PLAN_ROWS = 2048;
constexpr int TILE = 128;                          // columns that a block takes
constexpr int SIZES = 8;                           // sizes of an item that are looked at
constexpr int64_t MOST_KEYS = (int64_t)1 << 35;    // that tables have room for: sizes and 8 of them are 32 bits
// that a row's table has room for: up to 513 chunks of a row's keys, rounded up to 128, end within 32 bits
constexpr int64_t MOST_ROW = ((int64_t)1 << 31) - (1 << 20);

struct PlanSizes {
    int B, G, width, shift, tile, runs, max_units, max_slots;    // tile: members of TILE columns
};

__host__ __device__ constexpr int plan_units(int B) { return (PLAN_HEAD + 3 * B + 3) & ~3; }   // 16-byte aligned
__device__ __forceinline__ uint32_t cdiv(uint32_t a, uint32_t b) { return (a + b - 1) / b; }
__device__ __forceinline__ uint32_t in_sizes(int keys) { return ((uint32_t)keys + 63) >> 6; }
// chunks of a group's keys where an item has `run`, estimated; what a chunk has then; how many there are
__device__ __forceinline__ int about_chunks(int keys, float per_run) { return (int)ceilf(in_sizes(keys) * per_run); }
__device__ __forceinline__ int plan_chunk(int keys, float per_run) {
    return ((int)cdiv(keys, max(about_chunks(keys, per_run), 1)) + 127) & ~127;
}
__device__ __forceinline__ int plan_chunks(int keys, float per_run) {
    return keys > 0 ? (int)cdiv(keys, plan_chunk(keys, per_run)) : 0;
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void shared_plan_kernel(const int* __restrict__ seq_lens,
                                                              const int* __restrict__ leaders,
                                                              const int* __restrict__ shared,
                                                              int* __restrict__ plan, PlanSizes z) {
    constexpr int ROWS = THREADS == 1024 ? PLAN_ROWS : THREADS, NW = THREADS / WAVE;
    // of a row: keys, leader, keys behind the shared ones, place in the line, chunks of the shared
    // ones, first slot; of a leader: members, common keys, places in members and among the units
    __shared__ int keys[ROWS], lead[ROWS], rests[ROWS], chunks[ROWS], slot_of[ROWS], count[ROWS], common[ROWS],
        place[ROWS], unit_of[ROWS];
    __shared__ uint32_t line[ROWS], total[NW], items_of[SIZES];
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE, B = z.B;
    const int most = z.width << z.shift;
    auto wave_total = [](int v) { return __builtin_amdgcn_readlane(wave_sums(v), WAVE - 1); };
    for (int b = tid; b < B; b += THREADS) {
        keys[b] = min(max(seq_lens[b], 0), most);
        count[b] = 0;
        common[b] = INT32_MAX;
        place[b] = leaders[b];
    }
    __syncthreads();
    // a leader leads itself, and both have keys; any other row is its own
    for (int b = tid; b < B; b += THREADS) {
        const int l = place[b];
        const bool led = l >= 0 && l < B && l != b && place[l] == l && keys[b] > 0 && keys[l] > 0;
        const int to = lead[b] = led ? l : b, pages = keys[b] >> z.shift;
        atomicAdd(&count[to], 1);
        atomicMin(&common[to], led ? min(max(shared[b], 0), pages) : pages);
    }
    __syncthreads();
    // common becomes the keys that a leader's group shares
    int sum = 0;
    for (int b = tid; b < B; b += THREADS)
        if (lead[b] == b) {
            common[b] = count[b] > 1 ? common[b] << z.shift : 0;
            if (common[b]) sum += cdiv(count[b], z.tile) * (in_sizes(common[b]) + UNIT_COST);
        }
    __syncthreads();
    auto cost_of = [](int rest) { return rest > 0 ? in_sizes(rest) + UNIT_COST : 0u; };
    for (int b = tid; b < B; b += THREADS) {
        const int rest = rests[b] = keys[b] - common[lead[b]];
        sum += cost_of(rest);
    }
    sum = wave_total(sum);
    if (lane == 0) total[wave] = sum;
    __syncthreads();
    // the line
    uint32_t all = 0, behind = 0;
    for (int w = 0; w < NW; ++w) all += total[w];
    for (int b0 = 0; b0 < B; b0 += WAVE) {
        const int b = b0 + lane;
        const uint32_t mine = b < B ? cost_of(rests[b]) : 0, sums = wave_sums(mine);
        if (wave == 0 && b < B) line[b] = behind + sums - mine;
        behind += __builtin_amdgcn_readlane(sums, WAVE - 1);
    }
    // the smallest size that needs no more items than there are blocks, of those from an equal share to
    // one and a half times that
    const uint32_t share = max(2u, cdiv(all, (uint32_t)z.runs));
    auto size_of = [&](int i) { return share + share * i / (2 * SIZES); };
    for (int i = wave; i < SIZES; i += NW) {
        const uint32_t run = size_of(i);
        const float per_run = 1.0f / run;
        int n = 0;
        for (int b = lane; b < B; b += WAVE)
            if (common[b] > 0 && lead[b] == b) n += cdiv(count[b], z.tile) * about_chunks(common[b], per_run);
        n = wave_total(n);
        if (lane == 0) items_of[i] = n + cdiv(behind, run);
    }
    __syncthreads();
    int pick = 0;
    while (pick < SIZES - 1 && items_of[pick] > (uint32_t)z.runs) ++pick;
    const uint32_t run = size_of(pick);
    const float per_run = 1.0f / run;
    int* const first = plan + PLAN_HEAD;
    int* const splits = first + B;
    int* const members = splits + B;
    int* const units = plan + plan_units(B);
    // places of the groups' units and members
    int ahead = 0, at = 0;
    for (int b0 = 0; b0 < B; b0 += WAVE) {
        const int b = b0 + lane;
        int nu = 0, nm = 0;
        if (b < B && lead[b] == b) {
            const int n = plan_chunks(common[b], per_run);
            if (n) {
                nm = count[b];
                nu = (int)cdiv(nm, z.tile) * n;
            }
            if (wave == 0) chunks[b] = n;
        }
        const int iu = wave_sums(nu), im = wave_sums(nm);
        if (wave == 0 && b < B) {
            unit_of[b] = ahead + iu - nu;
            place[b] = at + im - nm;
        }
        ahead += __builtin_amdgcn_readlane(iu, WAVE - 1);
        at += __builtin_amdgcn_readlane(im, WAVE - 1);
    }
    // items of the line, and how much of it each has
    int lines = (int)cdiv(behind, run);
    if (behind > 0 && ahead + lines < z.runs) lines = (int)min((uint32_t)(z.runs - ahead), max(behind / 2, 1u));
    const uint32_t step = lines > 0 ? max(2u, cdiv(behind, lines)) : 1;
    if (lines > 0) lines = (int)cdiv(behind, step);
    const int items = ahead + lines;
    // Item i of the line begins where i * step falls, rounded to 128 keys of the row there: a row at
    // `line` is cut by the items that fall from line + 1 to the middle of its last 128 keys, and those
    // from there to the next row's first place begin with that row.
    auto cuts_from = [&](int b) { return (int)cdiv(line[b] + 1, step); };
    auto cuts_to = [&](int b) { return (int)cdiv(line[b] + 2 * ((uint32_t)(rests[b] + 127) >> 7) - 1, step); };
    auto cut = [&](int b, int i) { return (int)((i * step - line[b] + 1) >> 1 << 7); };
    __syncthreads();
    if (wave == 0) {
        int s = 0;
        for (int b0 = 0; b0 < B; b0 += WAVE) {
            const int b = b0 + lane;
            int ns = 0;
            if (b < B) {
                ns = chunks[lead[b]];
                if (rests[b] > 0) ns += 1 + cuts_to(b) - cuts_from(b);
            }
            const int is = wave_sums(ns);
            if (b < B) {
                first[b] = slot_of[b] = s + is - ns;
                splits[b] = ns;
            }
            s += __builtin_amdgcn_readlane(is, WAVE - 1);
        }
        if (lane == 0) {
            plan[0] = min(items, z.max_units);
            plan[1] = (int)behind;
        }
    }
    __syncthreads();
    auto write = [&](int u, int row, int k0, int k1, int place, int n, int split, int next) {
        if (u >= z.max_units) return;
        int4* d = reinterpret_cast<int4*>(units) + 2 * (size_t)u;
        d[0] = int4{row, k0, k1, place};
        d[1] = int4{n, split, next < z.max_units ? next : -1, row >= 0 ? slot_of[row] : 0};
    };
    // a wave a group, in turn: its members in order, and its units
    for (int r0 = 0, turn = 0; r0 < B; r0 += WAVE) {
        uint64_t groups = __ballot(r0 + lane < B && lead[min(r0 + lane, B - 1)] == r0 + lane && common[min(r0 + lane, B - 1)] > 0);
        for (; groups; groups &= groups - 1) {
            if (turn++ % NW != wave) continue;
            const int b = r0 + __builtin_ctzll(groups), p = common[b];
            for (int b0 = 0, m = place[b]; b0 < B; b0 += WAVE) {
                const bool mine = b0 + lane < B && lead[min(b0 + lane, B - 1)] == b;
                const uint64_t all_mine = __ballot(mine);
                if (mine) members[m + __builtin_popcountll(all_mine & ((1ull << lane) - 1))] = b0 + lane;
                m += __builtin_popcountll(all_mine);
            }
            const int c = plan_chunk(p, per_run), tiles = (int)cdiv(count[b], z.tile);
            for (int i = lane; i < chunks[b] * tiles; i += WAVE) {
                const int part = i / tiles, from = i % tiles * z.tile;
                write(unit_of[b] + i, b, part * c, min(part * c + c, p), place[b] + from, min(z.tile, count[b] - from), part, -1);
            }
        }
    }
    // the unit behind a row's last one in its item: the next row's first, unless that begins an item
    auto after = [&](int b) {
        while (++b < B && rests[b] <= 0) {}
        return b;
    };
    auto link = [&](int b) {
        const int next = after(b);
        return next < B && cuts_from(next) == cuts_to(b) ? items + next : -1;
    };
    // a thread a row: its first unit, and the items that have none, of those that fall between the
    // last row's last cut and this one, or behind the last row
    for (int b = tid; b < B; b += THREADS) {
        const int rest = rests[b];
        if (rest <= 0) continue;
        int before = b - 1;
        while (before >= 0 && rests[before] <= 0) --before;
        const int from = before >= 0 ? cuts_to(before) : 0, own = cuts_from(b), to = cuts_to(b);
        for (int i = from; i < own - 1; ++i) write(ahead + i, -1, 0, 0, 0, 0, 0, -1);
        if (after(b) == B)
            for (int i = to; i < lines; ++i) write(ahead + i, -1, 0, 0, 0, 0, 0, -1);
        const int p = keys[b] - rest, n = chunks[lead[b]];
        write(from < own ? ahead + own - 1 : items + b, b, p, p + (own < to ? cut(b, own) : rest), 0, 0, n,
              own < to ? -1 : link(b));
    }
    // a thread an item of the line: the unit that it begins with, where that is not a row's first
    for (int i = tid; i < lines; i += THREADS) {
        int b = 0, end = B;                      // the last row that begins at or before it
        while (end - b > 1) {
            const int mid = (b + end) / 2;
            if (line[mid] <= (uint32_t)i * step) b = mid;
            else end = mid;
        }
        const int own = cuts_from(b), to = cuts_to(b);
        if (rests[b] <= 0 || i < own || i >= to) continue;
        const int p = keys[b] - rests[b];
        write(ahead + i, b, p + cut(b, i), p + (i + 1 < to ? cut(b, i + 1) : rests[b]), 0, 0, chunks[lead[b]] + 1 + i - own,
              i + 1 < to ? -1 : link(b));
    }
}

// ---- attention ---------------------------------------------------------------------------------
struct SharedArgs {
    const char *q, *kc, *vc;
    const int *block_table, *seq_lens, *leaders, *shared;
    int* plan;
    float *o_part, *ml_part;
    int64_t q_row, q_head, k_page, k_token, k_head, v_page, v_token, v_head;     // bytes
    int64_t table_row;
    int B, Hq, Hk, G, pages, shift, slots;
    float scale;                                                                 // times log2(e)
    PlanSizes z;
    // Whether the rows' own keys are more than stays in the last cache until the next step, half of its
    // 256 MB: then they are read without being kept. 48 rows of up to 2000 tokens (197 MB) 50.4 -> 42.5
    // us, 64 of up to 512 (67 MB) 20.1 -> 21.2.
    int64_t size_bytes;                                                          // of 64 keys and values
    __device__ bool much(int sizes) const { return sizes * size_bytes >= (int64_t)128 << 20; }
};

constexpr int IDS = 1024;                          // pages of a unit that lie in LDS at a time

// what a block keeps in LDS of its item: the pages of a unit's keys; rows and slots of a group's tile;
// of a plan made here, the first unit and each row's first unit
struct SharedPlaces {
    int ids[IDS], rows[TILE], slots[TILE];
};
struct OwnPlan {
    int4 first[2];                                 // row (-1: none), first key, end, members |
                                                   // slot, next row, items, sizes of the line
    int4 row[WAVE];                                // first key, end, slot, next row
    int count[WAVE], common[WAVE];
};

// The plan of up to 64 rows, as shared_plan_kernel makes it, by one wave for itself: a lane a row. A
// call takes 1.1 to 1.9 us more than with a plan made before; a launch that makes one takes 8 for 128
// rows, and is what a step of many layers does once.
__device__ __forceinline__ void plan_item(const SharedArgs& a, int item, OwnPlan& own, SharedPlaces& places) {
    const PlanSizes& z = a.z;
    int lane = threadIdx.x & (WAVE - 1);
    asm volatile("" : "+v"(lane));                           // nothing of this is kept meanwhile
    const int B = z.B;
    const bool in = lane < B;
    const int most = z.width << z.shift;
    const int keys = in ? min(max(a.seq_lens[lane], 0), most) : 0;
    const int l = in ? a.leaders[lane] : lane, sh = in ? a.shared[lane] : 0;
    own.count[lane] = 0;
    own.common[lane] = INT32_MAX;
    const int l_of = __shfl(l, l & (WAVE - 1), WAVE), l_keys = __shfl(keys, l & (WAVE - 1), WAVE);
    const bool led = in && (uint32_t)l < (uint32_t)B && l != lane && l_of == l && keys > 0 && l_keys > 0;
    const int to = led ? l : lane, pages = keys >> z.shift;
    atomicAdd(&own.count[to], 1);
    atomicMin(&own.common[to], led ? min(max(sh, 0), pages) : pages);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int count = own.count[lane], common = count > 1 ? own.common[lane] << z.shift : 0;
    const int tiles = (int)cdiv(count, z.tile);
    const int p = __shfl(common, to, WAVE), rest = keys - p;
    auto wave_total = [](int v) { return __builtin_amdgcn_readlane(wave_sums(v), WAVE - 1); };
    const uint32_t cost = rest > 0 ? in_sizes(rest) + UNIT_COST : 0, sums = wave_sums(cost), line = sums - cost;
    const uint32_t behind = __builtin_amdgcn_readlane(sums, WAVE - 1);
    const uint32_t all = behind + wave_total(common ? tiles * (in_sizes(common) + UNIT_COST) : 0);
    const uint32_t share = max(2u, cdiv(all, (uint32_t)z.runs));
    uint32_t run = share;
    for (int i = 0; i < SIZES; ++i) {
        run = share + share * i / (2 * SIZES);
        const int n = wave_total(common ? tiles * about_chunks(common, 1.0f / run) : 0);
        if (n + cdiv(behind, run) <= (uint32_t)z.runs) break;
    }
    const float per_run = 1.0f / run;
    const int chunk = common ? plan_chunk(common, per_run) : 1, chunks = common ? (int)cdiv(common, chunk) : 0;
    const int nu = tiles * chunks, iu = wave_sums(nu), unit_of = iu - nu, ahead = __builtin_amdgcn_readlane(iu, WAVE - 1);
    int lines = (int)cdiv(behind, run);
    if (behind > 0 && ahead + lines < z.runs) lines = (int)min((uint32_t)(z.runs - ahead), max(behind / 2, 1u));
    const uint32_t step = lines > 0 ? max(2u, cdiv(behind, lines)) : 1;
    if (lines > 0) lines = (int)cdiv(behind, step);
    const int from = (int)cdiv(line + 1, step);
    const int upto = rest > 0 ? (int)cdiv(line + 2 * ((uint32_t)(rest + 127) >> 7) - 1, step) : 0;
    auto cut = [&](int i) { return (int)((i * step - line + 1) >> 1 << 7); };
    const int shared_chunks = __shfl(chunks, to, WAVE);
    const int splits = shared_chunks + (rest > 0 ? 1 + upto - from : 0), slot = wave_sums(splits) - splits;
    if (blockIdx.x == 0 && in) {                             // for the combine
        a.plan[PLAN_HEAD + lane] = slot;
        a.plan[PLAN_HEAD + B + lane] = splits;
    }
    const uint64_t live = __ballot(rest > 0), below = live & ((1ull << lane) - 1), above = live & ~((2ull << lane) - 1);
    const int ended = __shfl(upto, below ? 63 - __builtin_clzll(below) : 0, WAVE), before = below ? ended : 0;
    const int next = above ? __builtin_ctzll(above) : 0, next_from = __shfl(from, next, WAVE);
    const int link = above && next_from == upto ? next : -1;
    const int start = p + (from < upto ? cut(from) : rest), start_link = from < upto ? -1 : link;
    own.row[lane] = int4{p, start, slot + shared_chunks, start_link};
    if (lane == 0) own.first[0] = int4{-1, 0, 0, 0};
    if (lane == 0) own.first[1] = int4{0, -1, ahead + lines, (int)behind};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (item < ahead) {
        const int lead = __builtin_ctzll(__ballot(unit_of <= item && item < unit_of + nu));
        auto of_lead = [&](int v) { return __builtin_amdgcn_readlane(v, lead); };
        const int i = item - of_lead(unit_of), n = of_lead(tiles), part = i / n, at = i % n * z.tile, c = of_lead(chunk);
        const int members = min(z.tile, of_lead(count) - at);
        const bool mine = in && to == lead;
        const uint64_t all_mine = __ballot(mine);
        const int rank = __builtin_popcountll(all_mine & ((1ull << lane) - 1)) - at;
        if (mine && rank >= 0 && rank < members) {
            places.rows[rank] = lane;
            places.slots[rank] = slot + part;
        }
        if (lane == lead) own.first[0] = int4{lead, part * c, min(part * c + c, common), members};
    } else {
        const int i = item - ahead;
        if (rest > 0 && i == from - 1 && before < from) {
            own.first[0] = int4{lane, p, start, 0};
            own.first[1] = int4{slot + shared_chunks, start_link, ahead + lines, (int)behind};
        } else if (rest > 0 && i >= from && i < upto) {
            own.first[0] = int4{lane, p + cut(i), p + (i + 1 < upto ? cut(i + 1) : rest), 0};
            own.first[1] = int4{slot + shared_chunks + 1 + i - from, i + 1 < upto ? -1 : link, ahead + lines, (int)behind};
        }
    }
}

struct SharedUnit {
    int row, begin, end, group, slot, columns;     // group: members, their rows and slots in LDS
    bool once;                                     // keys that no cache holds until the next step
};
// Four waves take a unit's chunk for one key head. A wave has up to 32 columns (MT tiles of 16), so
// KG groups of waves share the keys out, 32 in turn, and the 4 / KG waves of a group the columns:
//     columns     up to 32     64     128
//     KG                 4      2       1
// Keys straight into registers, one wave a SIMD with 64 columns, took 562 us where this takes 116 (128 rows
// of 64 heads on 8 behind 16400 tokens); a ring of four steps of 32 keys for 128 columns, with the next step's
// products beside the weights, 163 where two of 64 took 122.
// Keys are the rows of the first product (S^T = K Q^T: a lane has the scores of one column, four keys
// of every sixteen), and the contraction of the second (O^T = V^T P^T) takes a lane's own weights as
// they are, keys 4g..+3 and 16 + 4g..+3 for lane group g; the transposing LDS read gives the values
// in the same order.
//
// Keys and values come by 16-byte transfers into LDS, 16 KiB a step of 32 keys and 128 channels, and
// a group has a ring of 4 / KG steps. A group of one wave asks for the next keys while it works on
// the values and for the next values behind that, with no barrier; the others have one a step. Two
// blocks fit a CU (LDS), so that one's ends and barriers are the other's work.
//
// 16-byte pieces of key rows and 32-byte pieces of value rows change places with the key, so that
// neither the reads of key rows nor the transposing ones meet in a bank; a transfer writes LDS in
// lane order, so its source address carries the change.
template <int N>
__device__ __forceinline__ void wait_transfers() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

__device__ __forceinline__ const char* same_in_wave(const char* p) {
    const uint64_t v = (uint64_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (const char*)((uint64_t)hi << 32 | lo);
}

// maximum over the four lane groups
__device__ __forceinline__ float over_groups(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <bool F16, int D, int MT, int KG>
__device__ __forceinline__ void shared_unit(const SharedArgs& a, const SharedUnit& unit, int h, char* lds, SharedPlaces& places) {
    constexpr int NS = D / 32, ND = D / 16, ROW = D * 2, CPR = ROW / 16;
    constexpr int CG = 4 / KG, KEYS = KG == 1 ? 64 : 32, STAGES = KG == 4 ? 1 : 2;
    constexpr int PLANE = KEYS * ROW, STAGE = 2 * PLANE, NJ = KEYS / 16;
    constexpr int RPP = 1024 / ROW, PCS = 32 / RPP;          // rows of a transfer, transfers of 32 rows
    constexpr int COLS = CG * 32;
    constexpr float LARGEST = F16 ? 15.0f : 0.0f;
    int lane = threadIdx.x & (WAVE - 1);
    asm volatile("" : "+v"(lane));           // places in LDS are worked out here, not kept from unit to unit
    const int col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int kg = wave / CG, cg = wave % CG;
    const int row0 = unit.row, begin = unit.begin, end = unit.end, columns = unit.columns;
    const int G = a.G, mask = (1 << a.shift) - 1;
    constexpr int RING = 4 * 32 * D * 4;
    int* const ids = places.ids;
    char* const ring = lds + kg * (RING / KG);
    const uint32_t ring_at = (uint32_t)(uintptr_t)ring;

    uint4 qf[MT][NS];
    const bool busy = cg * 32 < columns;                     // the wave has columns
    // signs of q so that larger products are larger weights; no q at all where the scale is 0
    const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u, keep_q = a.scale == 0.0f ? 0u : ~0u;
    const float scale = a.scale == 0.0f ? 1.0f : fabsf(a.scale);
    auto load_q = [&](bool group) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int c = cg * 32 + m * 16 + col;
            const bool in = c < columns;
            const int cc = in ? c : 0;
            const char* at = group ? a.q + places.rows[cc / G] * a.q_row + (h * G + cc % G) * a.q_head + g * 16
                                   : a.q + row0 * a.q_row + (h * G + cc) * a.q_head + g * 16;
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                const uint4 w = *reinterpret_cast<const uint4*>(at + s * 64);
                qf[m][s] = in ? uint4{(w.x ^ flip) & keep_q, (w.y ^ flip) & keep_q, (w.z ^ flip) & keep_q, (w.w ^ flip) & keep_q}
                              : uint4{0, 0, 0, 0};
            }
        }
    };
    if (!unit.group) load_q(false);                          // a group's rows are known behind the barrier
    sh_f4 o[MT][ND];
    // sums of weights come from the matrix cores too, as the product with values of 1: of the rounded
    // weights, which the outputs are made of
    sh_f4 sum[MT];
    float mx[MT];
    const uint32_t one = F16 ? 0x3c003c00u : 0x3f803f80u;
    const uint4 ones = {one, one, one, one};
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        mx[m] = -INFINITY;
        sum[m] = sh_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int d = 0; d < ND; ++d) o[m][d] = sh_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const char* const kb = a.kc + h * a.k_head;
    const char* const vb = a.vc + h * a.v_head;
    auto swz_k = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
    auto swz_v = [](int r) { return D == 128 ? r & 7 : (r >> 1) & 3; };

    // the unit's keys in spans whose pages lie in LDS; what a table should not hold reads the last page
    const int span = (int)min((int64_t)(IDS - 16) << a.shift & ~(int64_t)127, (int64_t)1 << 30);
    int k0 = begin, k1 = begin + min(span, end - begin), page0 = k0 >> a.shift;
    auto place_pages = [&]() {
        const int* const table = a.block_table + row0 * a.table_row;
        page0 = k0 >> a.shift;
        for (int i = threadIdx.x; i <= ((k1 - 1) >> a.shift) - page0; i += 256)
            ids[i] = (int)min((uint32_t)table[page0 + i], (uint32_t)(a.pages - 1));
    };
    place_pages();
    // 32 rows of keys or values from `key` on. What lies past the chunk is its last key, so that
    // nothing that no row owns is read.
    const int r_lane = lane / CPR, pc = lane % CPR;
    auto load_rows = [&](bool values, int key, uint32_t to) {
        key = __builtin_amdgcn_readfirstlane(key);
        to = __builtin_amdgcn_readfirstlane(to);
        const char* const base = values ? vb : kb;
        const int64_t step = values ? a.v_page : a.k_page;
        const int token = (int)(values ? a.v_token : a.k_token);
        const int last = k1 - 1 - key;
        auto place_of = [&](int p, int& at) {                // in the row; and the row
            const int r = p * RPP + r_lane;
            at = min(r, last);
            return (values ? (((pc >> 1) ^ swz_v(r)) << 1 | (pc & 1)) : pc ^ swz_k(r)) * 16;
        };
        if (a.shift >= 5) {                                  // rows of one page
            const int page = __builtin_amdgcn_readfirstlane(ids[(key >> a.shift) - page0]);
            const char* const rows = same_in_wave(base + page * step + (int64_t)(key & mask) * token);
#pragma unroll
            for (int p = 0; p < 32 / RPP; ++p) {
                int at;
                const int place = place_of(p, at);
                if (KG == 4 && unit.once) lds_transfer16<true>(to + p * 1024, __umul24(at, token) + place, rows);
                else lds_transfer16(to + p * 1024, __umul24(at, token) + place, rows);
            }
        } else {
#pragma unroll
            for (int p = 0; p < 32 / RPP; ++p) {
                int at;
                const int place = place_of(p, at), kk = key + at;
                lds_transfer16(to + p * 1024, base + ids[(kk >> a.shift) - page0] * step + (int64_t)(kk & mask) * token + place);
            }
        }
    };

    // a step's keys from LDS: scores, weights, and their product with the values
    uint4 pf[MT][NJ / 2];
    sh_f4 sc[MT][NJ];
    auto products = [&](const char* kt) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            uint4 kf[NS];
#pragma unroll
            for (int s = 0; s < NS; ++s)
                kf[s] = *reinterpret_cast<const uint4*>(kt + (j * 16 + col) * ROW + ((s * 4 + g) ^ swz_k(j * 16 + col)) * 16);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                sc[m][j] = sh_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < NS; ++s) sc[m][j] = sh_product<F16>(kf[s], qf[m][s], sc[m][j]);
            }
        }
    };
    // values behind the chunk's last key are copies of its, and an infinite one times a weight of 0 would be
    // no number. Waves that share a step all write the same zeros, each before it reads.
    auto clear_behind = [&](char* vt, int key) {
        int from = (int)threadIdx.x & (WAVE - 1);
        asm volatile("" : "+v"(from));                       // nothing of this is kept meanwhile
#pragma unroll 1
        for (int at = (k1 - key) * ROW + from * 16; at < KEYS * ROW; at += 1024) *reinterpret_cast<uint4*>(vt + at) = uint4{0, 0, 0, 0};
    };
    // the largest weight is 2^LARGEST
    auto top_of = [&](float mx) { return mx * scale - LARGEST; };
    auto weights = [&](int key, char* vt) {
        if (key + KEYS > k1) {
            asm volatile("" : : : "memory");                 // a branch: every other step goes without
            if (KG < 4) clear_behind(vt, key);
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (key + j * 16 + g * 4 + r >= k1)
#pragma unroll
                        for (int m = 0; m < MT; ++m) sc[m][j][r] = -INFINITY;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float top = sc[m][0][0];
#pragma unroll
            for (int i = 1; i < NJ * 4; ++i) top = fmaxf(top, sc[m][i >> 2][i & 3]);
            top = over_groups(top);
            if (__any(top > mx[m])) {
                const float now = fmaxf(top, mx[m]);
                const float keep = mx[m] == now ? 1.0f : __builtin_amdgcn_exp2f((mx[m] - now) * scale);
                mx[m] = now;
#pragma unroll
                for (int r = 0; r < 4; ++r) sum[m][r] *= keep;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[m][d][r] *= keep;
            }
            const float base = mx[m] == -INFINITY ? 0.0f : top_of(mx[m]);
#pragma unroll
            for (int i = 0; i < NJ * 4; ++i)
                sc[m][i >> 2][i & 3] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[m][i >> 2][i & 3], scale, -base));
#pragma unroll
            for (int j = 0; j < NJ; j += 2)
                pf[m][j / 2] = uint4{sh_pack<F16>(sc[m][j][0], sc[m][j][1]), sh_pack<F16>(sc[m][j][2], sc[m][j][3]),
                                     sh_pack<F16>(sc[m][j + 1][0], sc[m][j + 1][1]),
                                     sh_pack<F16>(sc[m][j + 1][2], sc[m][j + 1][3])};
        }
    };
    auto value = [&](const char* vt, int half, int d) {
        union {
            struct { sh_s4 lo, hi; } p;
            uint4 u;
        } v;
        const int r = half * 32 + g * 4 + (col >> 2);
        const char* lo = vt + r * ROW + (d ^ swz_v(r)) * 32 + (col & 3) * 8;
        const char* hi = vt + (r + 16) * ROW + (d ^ swz_v(r + 16)) * 32 + (col & 3) * 8;
        v.p.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sh_s4*)lo);
        v.p.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sh_s4*)hi);
        return v.u;
    };
    // reads are three products ahead of their use: without a fixed order the compiler waits for each (128
    // rows of 64 heads on 8 behind 16400 tokens 125 us; one ahead 117, two 118, three 116, four 121)
    auto add_values = [&](const char* vt) {
        constexpr int AHEAD = 3, ALL = NJ / 2 * ND;
        uint4 v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) v[i] = value(vt, i / ND, i % ND);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < ALL; ++i) {
            const int half = i / ND, d = i % ND;
            const uint4 now = v[i % AHEAD];
            if (i + AHEAD < ALL) v[i % AHEAD] = value(vt, (i + AHEAD) / ND, (i + AHEAD) % ND);
            if (d == 0)
#pragma unroll
                for (int m = 0; m < MT; ++m) sum[m] = sh_product<F16>(ones, pf[m][half], sum[m]);
#pragma unroll
            for (int m = 0; m < MT; ++m) o[m][d] = sh_product<F16>(now, pf[m][half], o[m][d]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    __syncthreads();                                         // the places
    if (unit.group) load_q(true);
    for (;;) {
    if constexpr (KG == 4) {
        int key = k0 + kg * 32;
        if (key < k1) {
            load_rows(false, key, ring_at);
            load_rows(true, key, ring_at + PLANE);
        }
        for (; key < k1; key += 128) {
            wait_transfers<PCS>();
            products(ring);
            wait_reads();
            const bool more = key + 128 < k1;
            if (more) load_rows(false, key + 128, ring_at);
            weights(key, ring + PLANE);
            if (more) wait_transfers<PCS>();
            else {
                wait_transfers<0>();
                if (key + KEYS > k1) clear_behind(ring + PLANE, key);
            }
            add_values(ring + PLANE);
            wait_reads();
            if (more) load_rows(true, key + 128, ring_at + PLANE);
        }
    } else {
        // a wave brings 32 rows of a step: the first waves keys, the others values
        static_assert(CG * 32 == 2 * KEYS, "as many waves as there are 32 rows");
        // steps of the block, and of this group
        const int steps = CEIL_DIV(k1 - k0, KEYS * KG), mine = CEIL_DIV(k1 - k0 - kg * KEYS, KEYS * KG);
        auto key_of = [&](int i) { return k0 + (i * KG + kg) * KEYS; };
        auto ask = [&](int i) {
            const int half = cg % (KEYS / 32) * 32, key = key_of(i) + half;
            const bool values = cg >= KEYS / 32;
            // a step's second half may lie past the chunk: any rows of it do
            if (i < mine)
                load_rows(values, key < k1 ? key : key - half, ring_at + i % STAGES * STAGE + (values ? PLANE : 0) + half * ROW);
        };
        ask(0);
        for (int i = 0; i < steps; ++i) {
            // this step has come, and nobody is at the one before
            wait_transfers<0>();
            wait_reads();
            asm volatile("s_barrier" : : : "memory");
            ask(i + 1);
            char* const at = ring + i % STAGES * STAGE;
            if (busy && i < mine) {
                products(at);
                weights(key_of(i), at + PLANE);
                add_values(at + PLANE);
            }
        }
    }
    if (k1 >= end) break;
    __syncthreads();                                         // all have read the span's pages
    k0 = k1;
    k1 = k0 + min(span, end - k0);
    place_pages();
    __syncthreads();
    }

    if constexpr (KG == 1) {                                 // a column's sums are one wave's
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int c = cg * 32 + m * 16 + col;
            if (c >= columns) continue;
            const int slot = unit.group ? places.slots[c / G] : unit.slot;
            if (slot >= a.slots) continue;
            const size_t to = (size_t)slot * a.Hq + h * G + c % G;
#pragma unroll
            for (int d = 0; d < ND; ++d) *reinterpret_cast<sh_f4*>(a.o_part + to * D + d * 16 + g * 4) = o[m][d];
            if (g == 0)
                *reinterpret_cast<float2*>(a.ml_part + to * 2) =
                    float2{mx[m] == -INFINITY ? -INFINITY : top_of(mx[m]), sum[m][0]};
        }
        return;
    }
    // a common maximum of the groups' sums of each column, in units of the weights' exponent
    __syncthreads();
    constexpr int PITCH = D + 4;
    float* const merge = reinterpret_cast<float*>(lds);                       // [KG][COLS][PITCH]
    float* const stats = merge + KG * COLS * PITCH;                           // [KG][COLS][2]
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int c = cg * 32 + m * 16 + col;
        if (c >= columns) continue;
        if (g == 0)
            *reinterpret_cast<float2*>(stats + (kg * COLS + c) * 2) =
                float2{mx[m] == -INFINITY ? -INFINITY : top_of(mx[m]), sum[m][0]};
#pragma unroll
        for (int d = 0; d < ND; ++d)
            *reinterpret_cast<sh_f4*>(merge + (kg * COLS + c) * PITCH + d * 16 + g * 4) = o[m][d];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < columns * (D / 4); i += 256) {
        const int c = i / (D / 4), ch = i % (D / 4) * 4;
        float2 st[KG];
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < KG; ++w) {
            st[w] = *reinterpret_cast<const float2*>(stats + (w * COLS + c) * 2);
            top = fmaxf(top, st[w].x);
        }
        float l = 0.0f;
        sh_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < KG; ++w) {
            const float f = st[w].x == top ? 1.0f : __builtin_amdgcn_exp2f(st[w].x - top);
            l += st[w].y * f;
            acc += *reinterpret_cast<const sh_f4*>(merge + (w * COLS + c) * PITCH + ch) * f;
        }
        const int slot = unit.group ? places.slots[c / G] : unit.slot;
        if (slot >= a.slots) continue;
        const size_t to = (size_t)slot * a.Hq + h * G + c % G;
        *reinterpret_cast<sh_f4*>(a.o_part + to * D + ch) = acc;
        if (ch == 0) *reinterpret_cast<float2*>(a.ml_part + to * 2) = float2{top, l};
    }
}

// Grid: `runs` blocks for each key head, the heads of an item side by side: with eight of them a key
// head is on one die, whose L2 then has a chunk for all tiles of columns. PLANNED: by a plan made
// before; else of up to 64 rows, by one that the block makes.
template <bool F16, int D, bool PLANNED>
__global__ __launch_bounds__(256, 2) void shared_attn_kernel(SharedArgs a) {
    constexpr int RING = 4 * 32 * D * 4, MERGE = 4 * 32 * (D + 4 + 2) * 4;
    __shared__ __attribute__((aligned(16))) char lds[RING > MERGE ? RING : MERGE];
    __shared__ SharedPlaces places;
    const int h = blockIdx.x % a.Hk, begin = blockIdx.x / a.Hk;
    auto same = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    auto take = [&](const SharedUnit& unit) {
        if (unit.columns <= 16) shared_unit<F16, D, 1, 4>(a, unit, h, lds, places);
        else if (unit.columns <= 32) shared_unit<F16, D, 2, 4>(a, unit, h, lds, places);
        else if (unit.columns <= 64) shared_unit<F16, D, 2, 2>(a, unit, h, lds, places);
        else shared_unit<F16, D, 2, 1>(a, unit, h, lds, places);
        __syncthreads();                                     // LDS is the next unit's
    };
    if constexpr (PLANNED) {
        const int* const first = a.plan + PLAN_HEAD;
        const int* const members = first + 2 * a.B;
        const int4* const units = reinterpret_cast<const int4*>(a.plan + plan_units(a.B));
        // the number of items and the first one's record in one wait: there is room for `runs` of them
        const int count = a.plan[0], behind = a.plan[1];
        int4 x = units[2 * (size_t)begin], y = units[2 * (size_t)begin + 1];
        const int items = same(count);
        const bool once = a.much(same(behind));
        for (int i = begin; i < items; i += a.z.runs)
            for (int u = i; u >= 0;) {
                if (u != begin) {
                    x = units[2 * (size_t)u];
                    y = units[2 * (size_t)u + 1];
                }
                const int place = same(x.w), split = same(y.y);
                SharedUnit unit = {same(x.x), same(x.y), same(x.z), same(y.x), same(y.w) + split, 0, !same(y.x) && once};
                unit.columns = max(unit.group, 1) * a.G;
                u = same(y.z);
                if ((uint32_t)unit.row >= (uint32_t)a.B) continue;   // an item without units
                for (int j = threadIdx.x; j < unit.group; j += 256) {
                    const int b = members[place + j];
                    places.rows[j] = b;
                    places.slots[j] = first[b] + split;
                }
                take(unit);
            }
    } else {
        __shared__ OwnPlan own;
        for (int i = begin;; i += a.z.runs) {
            if (threadIdx.x < WAVE) plan_item(a, i, own, places);
            __syncthreads();
            int4 x = own.first[0];
            const int4 y = own.first[1];
            const int items = same(y.z);
            const bool once = a.much(same(y.w));
            SharedUnit unit = {same(x.x), same(x.y), same(x.z), same(x.w), same(y.x), 0, !same(x.w) && once};
            unit.columns = max(unit.group, 1) * a.G;
            for (int next = same(y.y); (uint32_t)unit.row < (uint32_t)a.B;) {
                take(unit);
                if (next < 0) break;
                x = own.row[next];
                unit = SharedUnit{next, same(x.x), same(x.y), 0, same(x.z), a.G, once};
                next = same(x.w);
            }
            if (i + a.z.runs >= items) break;
            __syncthreads();                                 // all have read the item
        }
    }
}

// PER waves take a (row, head): the slots' sums with their common maximum. Weights of up to 64 slots
// are worked out by a lane each; sums are read eight at a time.
template <bool F16, int D, int PER>
__global__ __launch_bounds__(256) void shared_combine_kernel(const float* __restrict__ o_part,
                                                             const float* __restrict__ ml_part,
                                                             const int* __restrict__ plan, char* __restrict__ out,
                                                             int B, int Hq, int slots) {
    constexpr int CH = D / WAVE;
    __shared__ float red[4][D + 2];
    const int lane = threadIdx.x & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int pair = blockIdx.x * (4 / PER) + wave / PER, part = wave % PER;
    if (pair >= B * Hq) return;                              // with PER > 1 all of a block or none
    const int b = pair / Hq, h = pair % Hq;
    const int s0 = plan[PLAN_HEAD + b];
    const int n = min(plan[PLAN_HEAD + B + b], slots - s0);
    const float2* const ml = reinterpret_cast<const float2*>(ml_part) + (size_t)s0 * Hq + h;
    const float* const o = o_part + ((size_t)s0 * Hq + h) * D + lane * CH;
    float top = -INFINITY, acc[CH], total = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) acc[c] = 0.0f;
    const int parts = n > part ? CEIL_DIV(n - part, PER) : 0;         // slots part, part + PER, ...
    for (int b0 = 0; b0 < parts; b0 += WAVE) {
        const int here = min(parts - b0, WAVE);
        const float2 mine = lane < here ? ml[(size_t)((b0 + lane) * PER + part) * Hq] : float2{-INFINITY, 0.0f};
        const float now = fmaxf(top, wave_reduce_max(mine.x));
        const float base = now == -INFINITY ? 0.0f : now;
        const float keep = top == now ? 1.0f : __builtin_amdgcn_exp2f(top - base);
        const float f = mine.x == base ? 1.0f : __builtin_amdgcn_exp2f(mine.x - base);
        top = now;
        total = total * keep + wave_reduce_sum(mine.y * f);
#pragma unroll
        for (int c = 0; c < CH; ++c) acc[c] *= keep;
        for (int s = 0; s < here; s += 8) {
            float v[8][CH];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float* const at = o + (size_t)((b0 + min(s + i, here - 1)) * PER + part) * Hq * D;
                if constexpr (CH == 2) {
                    const float2 w = *reinterpret_cast<const float2*>(at);
                    v[i][0] = w.x;
                    v[i][1] = w.y;
                } else {
                    v[i][0] = *at;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float w = __shfl(f, min(s + i, here - 1), WAVE);
                if (s + i < here)
#pragma unroll
                    for (int c = 0; c < CH; ++c) acc[c] += v[i][c] * w;
            }
        }
    }
    if constexpr (PER > 1) {
#pragma unroll
        for (int c = 0; c < CH; ++c) red[wave][lane * CH + c] = acc[c];
        if (lane == 0) {
            red[wave][D] = top;
            red[wave][D + 1] = total;
        }
        __syncthreads();
        if (part) return;
        for (int w = 0; w < PER; ++w) top = fmaxf(top, red[w][D]);
        const float base = top == -INFINITY ? 0.0f : top;
        total = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c) acc[c] = 0.0f;
        for (int w = 0; w < PER; ++w) {
            const float f = red[w][D] == base ? 1.0f : __builtin_amdgcn_exp2f(red[w][D] - base);
            total += red[w][D + 1] * f;
#pragma unroll
            for (int c = 0; c < CH; ++c) acc[c] += red[w][lane * CH + c] * f;
        }
    }
    const float r = total == 0.0f ? 1.0f : total;
    if constexpr (CH == 2)
        reinterpret_cast<uint32_t*>(out)[(size_t)pair * WAVE + lane] = sh_pack<F16>(acc[0] / r, acc[1] / r);
    else
        reinterpret_cast<uint16_t*>(out)[(size_t)pair * WAVE + lane] = (uint16_t)sh_pack<F16>(acc[0] / r, 0.0f);
}

// ---- entries -----------------------------------------------------------------------------------
static bool shared_sizes(int B, int Hq, int Hk, int D) {
    return B >= 1 && B <= PLAN_ROWS && Hk >= 1 && Hq >= Hk && Hq % Hk == 0 && Hq <= 4096 && Hq / Hk <= TILE && (D == 64 || D == 128);
}

static bool table_sizes(int B, int width, int shift) {
    return (int64_t)B * width <= MOST_KEYS >> shift && width <= MOST_ROW >> shift;
}

// Blocks of a key head: two a CU. Units: items, of which there are at the most `runs` and one for each
// tile of a group (B / tile and one more for each of B / 2 groups) beside as many of the line, and one
// more a row. Slots: what an item of a tile leaves is a slot for each of its members, of which there
// are `tile` or B, and a row has one more of each kind than equal shares would make. Many rows of many heads
// on few take the most memory for them: 2048 of 128 on 1, of 128 channels, 0.6 GB.
static PlanSizes plan_sizes(int B, int Hq, int Hk, int width, int shift) {
    PlanSizes z;
    z.B = B;
    z.G = Hq / Hk;
    z.width = width;
    z.shift = shift;
    z.tile = max(1, TILE / z.G);
    z.runs = max(1, 512 / Hk);                               // 256, 768 or 1024 blocks in all: level or slower
    z.max_units = 2 * z.runs + B / z.tile + B / 2 + B + 16;
    z.max_slots = (min(z.tile, B) + 1) * z.runs + 4 * B + 16;
    return z;
}

// ints of a plan, and slots of partial results
extern "C" int oa_shared_plan_size(int B, int Hq, int Hk, int D, int* ints, int* slots) {
    if (!shared_sizes(B, Hq, Hk, D)) return -100;
    const PlanSizes z = plan_sizes(B, Hq, Hk, 1, 0);
    *ints = plan_units(B) + z.max_units * UNIT;
    *slots = z.max_slots;
    return 0;
}

static int launch_plan(hipStream_t stream, const void* seq_lens, const void* leaders, const void* shared, void* plan,
                       const PlanSizes& z) {
    if (z.B <= 256)
        hipLaunchKernelGGL(shared_plan_kernel<256>, dim3(1), dim3(256), 0, stream, (const int*)seq_lens,
                           (const int*)leaders, (const int*)shared, (int*)plan, z);
    else
        hipLaunchKernelGGL(shared_plan_kernel<1024>, dim3(1), dim3(1024), 0, stream, (const int*)seq_lens,
                           (const int*)leaders, (const int*)shared, (int*)plan, z);
    HIP_CHECK_LAUNCH();
    return 0;
}

static int shift_of(int block_size) {
    return block_size >= 1 && (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
}

extern "C" int oa_shared_plan(void* stream, const void* seq_lens, const void* leaders, const void* shared, void* plan,
                              int B, int Hq, int Hk, int D, int width, int block_size) {
    if (!shared_sizes(B, Hq, Hk, D) || width < 1) return -100;
    const int shift = shift_of(block_size);
    if (shift < 0) return -101;
    if (!table_sizes(B, width, shift)) return -102;
    if ((uintptr_t)plan % 16 != 0) return -103;
    return launch_plan((hipStream_t)stream, seq_lens, leaders, shared, plan, plan_sizes(B, Hq, Hk, width, shift));
}

// sizes: strides in elements (q row, q head; k page, token, head; v page, token, head; table row), then rows, heads,
// key heads, channels, table width, pages, block size and whether the type is float16. leaders, shared, seq_lens:
// null where `plan` is made already. scratch: floats, (D + 2) for each slot and head.
extern "C" int oa_attention_decode_shared(void* stream, const void* q, const void* kc, const void* vc,
                                          const void* block_table, const void* seq_lens, const void* leaders,
                                          const void* shared, void* plan, void* scratch, void* out,
                                          const int64_t* sizes, float scale) {
    const int64_t* const n = sizes + 9;
    for (int i = 0; i < 7; ++i)
        if (n[i] < 0 || n[i] > INT32_MAX) return -100;
    const int B = (int)n[0], Hq = (int)n[1], Hk = (int)n[2], D = (int)n[3], width = (int)n[4], pages = (int)n[5];
    const int shift = shift_of((int)n[6]);
    if (!shared_sizes(B, Hq, Hk, D) || width < 1 || pages < 1) return -100;
    if (shift < 0) return -101;
    if (!table_sizes(B, width, shift)) return -102;
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)plan | (uintptr_t)scratch) % 16 != 0) return -103;
    for (int i = 0; i < 8; ++i)
        if (sizes[i] % 8 != 0) return -103;
    // a token's step is 24 bits in a transfer's offset
    if (sizes[3] < 0 || sizes[3] >= (1 << 23) || sizes[6] < 0 || sizes[6] >= (1 << 23)) return -105;
    const PlanSizes z = plan_sizes(B, Hq, Hk, width, shift);
    const hipStream_t s = (hipStream_t)stream;
    const bool planned = !leaders || B > WAVE;
    if (leaders && planned) {
        const int rc = launch_plan(s, seq_lens, leaders, shared, plan, z);
        if (rc) return rc;
    }
    SharedArgs a;
    a.q = (const char*)q;
    a.kc = (const char*)kc;
    a.vc = (const char*)vc;
    a.block_table = (const int*)block_table;
    a.seq_lens = (const int*)seq_lens;
    a.leaders = (const int*)leaders;
    a.shared = (const int*)shared;
    a.plan = (int*)plan;
    a.z = z;
    a.size_bytes = (int64_t)64 * 2 * Hk * D * 2;
    a.o_part = (float*)scratch;
    a.ml_part = a.o_part + (size_t)z.max_slots * Hq * D;
    int64_t* const steps[8] = {&a.q_row, &a.q_head, &a.k_page, &a.k_token, &a.k_head, &a.v_page, &a.v_token, &a.v_head};
    for (int i = 0; i < 8; ++i) *steps[i] = sizes[i] * 2;
    a.table_row = sizes[8];
    a.B = B;
    a.Hq = Hq;
    a.Hk = Hk;
    a.G = Hq / Hk;
    a.pages = pages;
    a.shift = shift;
    a.slots = z.max_slots;
    a.scale = scale * 1.44269504088896340736f;
    // four waves a (row, head) while that leaves every CU with little to do
    const bool wide = B * Hq <= 1024;
    const dim3 grid(z.runs * Hk), merge(wide ? B * Hq : CEIL_DIV(B * Hq, 4)), block(256);
#define LAUNCH(F16, DV)                                                                                            \
    do {                                                                                                           \
        if (planned) hipLaunchKernelGGL((shared_attn_kernel<F16, DV, true>), grid, block, 0, s, a);                \
        else hipLaunchKernelGGL((shared_attn_kernel<F16, DV, false>), grid, block, 0, s, a);                       \
        HIP_CHECK_LAUNCH();                                                                                        \
        if (wide)                                                                                                  \
            hipLaunchKernelGGL((shared_combine_kernel<F16, DV, 4>), merge, block, 0, s, a.o_part, a.ml_part, a.plan, \
                               (char*)out, B, Hq, a.slots);                                                        \
        else                                                                                                       \
            hipLaunchKernelGGL((shared_combine_kernel<F16, DV, 1>), merge, block, 0, s, a.o_part, a.ml_part, a.plan, \
                               (char*)out, B, Hq, a.slots);                                                        \
        HIP_CHECK_LAUNCH();                                                                                        \
    } while (0)
    if (n[7]) {
        if (D == 64) LAUNCH(true, 64);
        else LAUNCH(true, 128);
    } else {
        if (D == 64) LAUNCH(false, 64);
        else LAUNCH(false, 128);
    }
#undef LAUNCH
    return 0;
}
