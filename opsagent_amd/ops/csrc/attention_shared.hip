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
// numbers of the cache's type, which is off by half a step of each weight and averages out over the
// keys; the output is rounded to the same type.
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
// PLAN, in ints: units, slots (2, padded to 8) | first[B] | splits[B] | members[B], rows group after
// group | units of 8: table row, first key, end, place of the group in members (-1: the table row
// alone), first column, columns, split, 0. A column is a (member, head of the key head) pair.
//
// Keys of all jobs, a group's counted once for each tile of columns, are cut in about `target` equal
// chunks; a job has as many of them as its keys need, of equal size, a multiple of 128.
constexpr int PLAN_HEAD = 8, UNIT = 8;
constexpr int PLAN_ROWS = 2048;

struct PlanSizes {
    int B, G, width, shift, tile, target, max_units, max_slots;
};

__device__ __forceinline__ int plan_chunk(int keys, int chunk) {
    const int n = CEIL_DIV(keys, chunk);
    return (CEIL_DIV(keys, n) + 127) & ~127;
}

__global__ __launch_bounds__(1024) void shared_plan_kernel(const int* __restrict__ seq_lens,
                                                           const int* __restrict__ leaders,
                                                           const int* __restrict__ shared,
                                                           int* __restrict__ plan, PlanSizes z) {
    __shared__ int keys[PLAN_ROWS], lead[PLAN_ROWS], count[PLAN_ROWS], common[PLAN_ROWS], place[PLAN_ROWS];
    __shared__ int total[16], chunk_all;
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE, B = z.B;
    const int most = (int)min((int64_t)z.width << z.shift, (int64_t)INT32_MAX - 4096);
    for (int b = tid; b < B; b += 1024) {
        keys[b] = min(max(seq_lens[b], 0), most);
        count[b] = 0;
        common[b] = INT32_MAX;
        lead[b] = leaders[b];
    }
    __syncthreads();
    // a leader leads itself, and both have keys; any other row is its own
    for (int b = tid; b < B; b += 1024) {
        const int l = lead[b];
        const bool led = l >= 0 && l < B && l != b && lead[l] == l && keys[b] > 0 && keys[l] > 0;
        place[b] = led ? l : b;
    }
    __syncthreads();
    for (int b = tid; b < B; b += 1024) lead[b] = place[b];
    __syncthreads();
    for (int b = tid; b < B; b += 1024) {
        const int l = lead[b];
        atomicAdd(&count[l], 1);
        atomicMin(&common[l], l == b ? keys[b] >> z.shift : min(max(shared[b], 0), keys[b] >> z.shift));
    }
    __syncthreads();
    // common: keys that a leader's group shares; and the keys of all jobs
    const int tiles1 = CEIL_DIV(z.G, z.tile);
    float all = 0.0f;
    for (int b = tid; b < B; b += 1024) {
        if (lead[b] == b) {
            common[b] = count[b] > 1 ? common[b] << z.shift : 0;
            all += (float)common[b] * CEIL_DIV(count[b] * z.G, z.tile);
        }
    }
    __syncthreads();
    for (int b = tid; b < B; b += 1024) all += (float)(keys[b] - common[lead[b]]) * tiles1;
    all = wave_reduce_sum(all);
    if (lane == 0) total[wave] = __float_as_int(all);
    __syncthreads();
    if (tid == 0) {
        float t = 0.0f;
        for (int w = 0; w < 16; ++w) t += __int_as_float(total[w]);
        const float c = fminf(ceilf(t / z.target), (float)(INT32_MAX / 2));
        chunk_all = max(((int)c + 127) & ~127, 128);
    }
    __syncthreads();
    const int chunk = chunk_all;
    // places: the first wave adds up units, members and slots over the rows
    int* const first = plan + PLAN_HEAD;
    int* const splits = first + B;
    int* const members = splits + B;
    int* const units = members + B;
    __shared__ int unit_of[PLAN_ROWS], member_of[PLAN_ROWS];
    if (wave == 0) {
        int u = 0, m = 0, s = 0;
        for (int b0 = 0; b0 < B; b0 += WAVE) {
            const int b = b0 + lane;
            int nu = 0, nm = 0, ns = 0;
            if (b < B) {
                const int l = lead[b], p = common[l], rest = keys[b] - p;
                if (p > 0) ns = CEIL_DIV(p, plan_chunk(p, chunk));
                if (l == b && p > 0) {
                    nm = count[b];
                    nu = ns * CEIL_DIV(count[b] * z.G, z.tile);
                }
                if (rest > 0) {
                    const int c = CEIL_DIV(rest, plan_chunk(rest, chunk));
                    ns += c;
                    nu += c * tiles1;
                }
            }
            int iu = nu, im = nm, is = ns;
#pragma unroll
            for (int d = 1; d < WAVE; d <<= 1) {
                const int a = __shfl_up(iu, d, WAVE), e = __shfl_up(im, d, WAVE), f = __shfl_up(is, d, WAVE);
                if (lane >= d) {
                    iu += a;
                    im += e;
                    is += f;
                }
            }
            if (b < B) {
                unit_of[b] = u + iu - nu;
                member_of[b] = m + im - nm;
                first[b] = s + is - ns;
                splits[b] = ns;
            }
            u += __shfl(iu, WAVE - 1, WAVE);
            m += __shfl(im, WAVE - 1, WAVE);
            s += __shfl(is, WAVE - 1, WAVE);
        }
        if (lane == 0) {
            plan[0] = min(u, z.max_units);
            plan[1] = s;
        }
    }
    __syncthreads();
    // a wave a row: members of its group in order, and its units
    for (int b = wave; b < B; b += 16) {
        const int l = lead[b], p = common[l], rest = keys[b] - p;
        int u = unit_of[b], done = 0;
        if (l == b && p > 0) {
            for (int b0 = 0, m = member_of[b]; b0 < B; b0 += WAVE) {
                const bool mine = b0 + lane < B && lead[b0 + lane] == b;
                const uint64_t all_mine = __ballot(mine);
                if (mine) members[m + __builtin_popcountll(all_mine & ((1ull << lane) - 1))] = b0 + lane;
                m += __builtin_popcountll(all_mine);
            }
            const int c = plan_chunk(p, chunk), columns = count[b] * z.G;
            const int n = CEIL_DIV(p, c), tiles = CEIL_DIV(columns, z.tile);
            for (int i = lane; i < n * tiles; i += WAVE) {
                if (u + i >= z.max_units) break;
                int* d = units + (size_t)(u + i) * UNIT;
                const int part = i / tiles, col = i % tiles * z.tile;
                d[0] = b;
                d[1] = part * c;
                d[2] = min(part * c + c, p);
                d[3] = member_of[b];
                d[4] = col;
                d[5] = min(z.tile, columns - col);
                d[6] = part;
                d[7] = 0;
            }
            u += n * tiles;
        }
        if (p > 0) done = CEIL_DIV(p, plan_chunk(p, chunk));
        if (rest > 0) {
            const int c = plan_chunk(rest, chunk), n = CEIL_DIV(rest, c);
            for (int i = lane; i < n * tiles1; i += WAVE) {
                if (u + i >= z.max_units) break;
                int* d = units + (size_t)(u + i) * UNIT;
                const int part = i / tiles1, col = i % tiles1 * z.tile;
                d[0] = b;
                d[1] = p + part * c;
                d[2] = min(p + part * c + c, keys[b]);
                d[3] = -1;
                d[4] = col;
                d[5] = min(z.tile, z.G - col);
                d[6] = done + part;
                d[7] = 0;
            }
        }
    }
}

// ---- attention ---------------------------------------------------------------------------------
struct SharedArgs {
    const char *q, *kc, *vc;
    const int* block_table;
    const int* plan;
    float *o_part, *ml_part;
    int64_t q_row, q_head, k_page, k_token, k_head, v_page, v_token, v_head;     // bytes
    int64_t table_row;
    int B, Hq, Hk, G, pages, shift, slots;
    float scale;                                                                 // times log2(e)
};

// A block takes the chunk of a unit for one key head, its four waves 32 keys in turn. Keys are the
// rows of the first product (S^T = K Q^T: a lane has the scores of one column, four keys of every
// sixteen), and the contraction of the second (O^T = V^T P^T) takes a lane's own weights as they
// are, keys 4g..+3 and 16 + 4g..+3 for lane group g; the transposing LDS read gives the values in
// the same order. MT: tiles of 16 columns.
template <bool F16, int D, int MT>
__device__ __forceinline__ void shared_unit(const SharedArgs& a, const int* __restrict__ unit, int h, char* lds) {
    constexpr int NS = D / 32, ND = D / 16, ROW = D * 2, PIECES = ROW / 16;
    const int lane = threadIdx.x & (WAVE - 1), col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const int row0 = unit[0], k0 = unit[1], k1 = unit[2], group = unit[3], c0 = unit[4], columns = unit[5];
    const int* const table = a.block_table + row0 * a.table_row;
    const int* const members = a.plan + PLAN_HEAD + 2 * a.B;
    const int G = a.G;

    uint4 qf[MT][NS];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int c = m * 16 + col;
        const bool in = c < columns;
        const int cc = in ? c0 + c : c0;
        const int b = group < 0 ? row0 : members[group + cc / G];
        const char* at = a.q + b * a.q_row + (h * G + cc % G) * a.q_head + g * 16;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const uint4 w = *reinterpret_cast<const uint4*>(at + s * 64);
            qf[m][s] = in ? w : uint4{0, 0, 0, 0};
        }
    }
    sh_f4 o[MT][ND];
    float mx[MT], sum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        mx[m] = -INFINITY;
        sum[m] = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[m][d] = sh_f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const char* const kb = a.kc + h * a.k_head;
    const char* const vb = a.vc + h * a.v_head;
    const int mask = (1 << a.shift) - 1;
    // keys past the chunk's end are its last one: what it has is read, nothing that no row owns
    auto page_of = [&](int key) { return min((uint32_t)table[key >> a.shift], (uint32_t)(a.pages - 1)); };
    char* const vt = lds + wave * (32 * ROW);
    // 32-byte pieces of a value row change places with the key, so that the 16 keys that one
    // transposing read gathers lie in all banks
    auto swz = [](int key) { return D == 128 ? key & 7 : (key >> 1) & 3; };

    for (int at = k0 + wave * 32; at < k1; at += 128) {
        uint4 kf[2][NS];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int key = min(at + j * 16 + col, k1 - 1);
            const char* p = kb + page_of(key) * a.k_page + (key & mask) * a.k_token + g * 16;
#pragma unroll
            for (int s = 0; s < NS; ++s) kf[j][s] = *reinterpret_cast<const uint4*>(p + s * 64);
        }
        uint4 vf[PIECES / 2];
#pragma unroll
        for (int t = 0; t < PIECES / 2; ++t) {
            const int piece = t * WAVE + lane, r = piece / PIECES, u = piece % PIECES;
            const int key = min(at + r, k1 - 1);
            const int src = ((u >> 1) ^ swz(r)) * 32 + (u & 1) * 16;
            vf[t] = *reinterpret_cast<const uint4*>(vb + page_of(key) * a.v_page + (key & mask) * a.v_token + src);
        }
#pragma unroll
        for (int t = 0; t < PIECES / 2; ++t) *reinterpret_cast<uint4*>(vt + (t * WAVE + lane) * 16) = vf[t];

        uint4 pf[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float w[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                sh_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < NS; ++s) acc = sh_product<F16>(kf[j][s], qf[m][s], acc);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    w[j * 4 + r] = at + j * 16 + g * 4 + r < k1 ? acc[r] * a.scale : -INFINITY;
            }
            float top = w[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) top = fmaxf(top, w[i]);
            top = fmaxf(top, __shfl_xor(top, 16, WAVE));
            top = fmaxf(top, __shfl_xor(top, 32, WAVE));
            if (__any(top > mx[m])) {
                const float now = fmaxf(top, mx[m]);
                const float old = mx[m] == now ? 1.0f : exp2f(mx[m] - now);
                mx[m] = now;
                sum[m] *= old;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[m][d][r] *= old;
            }
            const float base = mx[m] == -INFINITY ? 0.0f : mx[m];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = exp2f(w[i] - base);
                sum[m] += w[i];
            }
            pf[m] = uint4{sh_pack<F16>(w[0], w[1]), sh_pack<F16>(w[2], w[3]), sh_pack<F16>(w[4], w[5]),
                          sh_pack<F16>(w[6], w[7])};
        }
        // the wave's own values: written above, read below
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            union {
                struct { sh_s4 lo, hi; } p;
                uint4 u;
            } v;
            const int r = g * 4 + (col >> 2);
            const char* lo = vt + r * ROW + (d ^ swz(r)) * 32 + (col & 3) * 8;
            const char* hi = vt + (r + 16) * ROW + (d ^ swz(r + 16)) * 32 + (col & 3) * 8;
            v.p.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sh_s4*)lo);
            v.p.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sh_s4*)hi);
#pragma unroll
            for (int m = 0; m < MT; ++m) o[m][d] = sh_product<F16>(v.u, pf[m], o[m][d]);
        }
        __builtin_amdgcn_wave_barrier();
    }

    // the waves' sums: a common maximum of each column, then each wave's share of the channels
    __syncthreads();
    constexpr int PITCH = D + 4;
    float* const merge = reinterpret_cast<float*>(lds);                       // [4][MT * 16][PITCH]
    float* const stats = merge + 4 * MT * 16 * PITCH;                         // [4][MT * 16][2]
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        sum[m] += __shfl_xor(sum[m], 16, WAVE);
        sum[m] += __shfl_xor(sum[m], 32, WAVE);
        if (g == 0) {
            float* s = stats + (wave * MT * 16 + m * 16 + col) * 2;
            s[0] = mx[m];
            s[1] = sum[m];
        }
#pragma unroll
        for (int d = 0; d < ND; ++d)
            *reinterpret_cast<sh_f4*>(merge + (wave * MT * 16 + m * 16 + col) * PITCH + d * 16 + g * 4) = o[m][d];
    }
    __syncthreads();
    const int* const first = a.plan + PLAN_HEAD;
    for (int i = threadIdx.x; i < columns * (D / 4); i += 256) {
        const int c = i / (D / 4), ch = i % (D / 4) * 4;
        float ms[4], top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            ms[w] = stats[(w * MT * 16 + c) * 2];
            top = fmaxf(top, ms[w]);
        }
        const float base = top == -INFINITY ? 0.0f : top;
        float l = 0.0f;
        sh_f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = ms[w] == base ? 1.0f : exp2f(ms[w] - base);
            l += stats[(w * MT * 16 + c) * 2 + 1] * f;
            acc += *reinterpret_cast<const sh_f4*>(merge + (w * MT * 16 + c) * PITCH + ch) * f;
        }
        const int cc = c0 + c;
        const int b = group < 0 ? row0 : members[group + cc / G];
        const int slot = first[b] + unit[6];
        if (slot >= a.slots) continue;
        const size_t to = (size_t)slot * a.Hq + h * G + cc % G;
        *reinterpret_cast<sh_f4*>(a.o_part + to * D + ch) = acc;
        if (ch == 0) *reinterpret_cast<float2*>(a.ml_part + to * 2) = float2{top, l};
    }
}

// Grid: units times key heads, the heads of a unit side by side: with eight of them a key head is on
// one die, whose L2 then has a chunk for all tiles of columns.
template <bool F16, int D, int MT>
__global__ __launch_bounds__(256) void shared_attn_kernel(SharedArgs a) {
    constexpr int RING = 4 * 32 * D * 2, MERGE = 4 * MT * 16 * (D + 4 + 2) * 4;
    __shared__ __attribute__((aligned(16))) char lds[RING > MERGE ? RING : MERGE];
    const int u = blockIdx.x / a.Hk, h = blockIdx.x % a.Hk;
    if (u >= a.plan[0]) return;
    const int* unit = a.plan + PLAN_HEAD + 3 * a.B + (size_t)u * UNIT;
    if (MT > 1 && unit[5] <= 16) shared_unit<F16, D, 1>(a, unit, h, lds);
    else shared_unit<F16, D, MT>(a, unit, h, lds);
}

// A wave a (row, head): the slots' sums with their common maximum.
template <bool F16, int D>
__global__ __launch_bounds__(256) void shared_combine_kernel(const float* __restrict__ o_part,
                                                             const float* __restrict__ ml_part,
                                                             const int* __restrict__ plan, char* __restrict__ out,
                                                             int B, int Hq, int slots) {
    const int pair = blockIdx.x * 4 + threadIdx.x / WAVE, lane = threadIdx.x & (WAVE - 1);
    if (pair >= B * Hq) return;
    const int b = pair / Hq, h = pair % Hq;
    const int s0 = plan[PLAN_HEAD + b];
    const int n = min(plan[PLAN_HEAD + B + b], slots - s0);
    float top = -INFINITY;
    for (int s = lane; s < n; s += WAVE) top = fmaxf(top, ml_part[((size_t)(s0 + s) * Hq + h) * 2]);
    top = wave_reduce_max(top);
    const float base = top == -INFINITY ? 0.0f : top;
    constexpr int CH = D / WAVE;
    float acc[CH], total = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) acc[c] = 0.0f;
#pragma unroll 4
    for (int s = 0; s < n; ++s) {
        const size_t at = (size_t)(s0 + s) * Hq + h;
        const float2 ml = *reinterpret_cast<const float2*>(ml_part + at * 2);
        const float f = ml.x == base ? 1.0f : exp2f(ml.x - base);
        total += ml.y * f;
#pragma unroll
        for (int c = 0; c < CH; ++c) acc[c] += o_part[at * D + lane * CH + c] * f;
    }
    const float r = total == 0.0f ? 1.0f : total;
    if constexpr (CH == 2)
        reinterpret_cast<uint32_t*>(out)[(size_t)pair * WAVE + lane] = sh_pack<F16>(acc[0] / r, acc[1] / r);
    else
        reinterpret_cast<uint16_t*>(out)[(size_t)pair * WAVE + lane] = (uint16_t)sh_pack<F16>(acc[0] / r, 0.0f);
}

// ---- entries -----------------------------------------------------------------------------------
// Columns that a block takes, and chunks that the keys of a key head are cut in: about two blocks a CU.
static int shared_tiles(int B, int G) { return (int64_t)B * G <= 16 ? 1 : (int64_t)B * G <= 32 ? 2 : 4; }
static int shared_target(int Hk) { return max(1, 512 / Hk); }

static bool shared_sizes(int B, int Hq, int Hk, int D) {
    return B >= 1 && B <= PLAN_ROWS && Hk >= 1 && Hq >= Hk && Hq % Hk == 0 && Hq <= 4096 && (D == 64 || D == 128);
}

// Units: chunks of `target` and one more for each job (rows, and a group's tiles of columns, of which
// there are at the most B * G / tile and one more for each of B / 2 groups). Slots: a chunk of a
// group's tile leaves tile / G of them, and every row has one more of each kind.
static PlanSizes plan_sizes(int B, int Hq, int Hk, int width, int shift) {
    PlanSizes z;
    z.B = B;
    z.G = Hq / Hk;
    z.width = width;
    z.shift = shift;
    z.tile = 16 * shared_tiles(B, z.G);
    z.target = shared_target(Hk);
    const int64_t tiles1 = CEIL_DIV(z.G, z.tile);
    z.max_units = (int)(z.target + (int64_t)B * z.G / z.tile + B / 2 + z.target + B * tiles1 + 8);
    z.max_slots = (int)((int64_t)z.tile * z.target / z.G + z.target + 2 * (int64_t)B + 8);
    return z;
}

// ints of a plan, and slots of partial results
extern "C" int oa_shared_plan_size(int B, int Hq, int Hk, int D, int* ints, int* slots) {
    if (!shared_sizes(B, Hq, Hk, D)) return -100;
    const PlanSizes z = plan_sizes(B, Hq, Hk, 1, 0);
    *ints = PLAN_HEAD + 3 * B + z.max_units * UNIT;
    *slots = z.max_slots;
    return 0;
}

extern "C" int oa_shared_plan(void* stream, const void* seq_lens, const void* leaders, const void* shared, void* plan,
                              int B, int Hq, int Hk, int D, int width, int block_size) {
    if (!shared_sizes(B, Hq, Hk, D) || width < 1) return -100;
    if (block_size < 1 || (block_size & (block_size - 1)) != 0) return -101;
    hipLaunchKernelGGL(shared_plan_kernel, dim3(1), dim3(1024), 0, (hipStream_t)stream, (const int*)seq_lens,
                       (const int*)leaders, (const int*)shared, (int*)plan,
                       plan_sizes(B, Hq, Hk, width, __builtin_ctz(block_size)));
    HIP_CHECK_LAUNCH();
    return 0;
}

// strides: q row, q head; k page, token, head; v page, token, head; table row: in elements
extern "C" int oa_attention_decode_shared(void* stream, const void* q, const void* kc, const void* vc,
                                          const void* block_table, const void* plan, void* o_part, void* ml_part,
                                          void* out, const int64_t* strides, int B, int Hq, int Hk, int D, int pages,
                                          int block_size, float scale, int f16) {
    if (!shared_sizes(B, Hq, Hk, D) || pages < 1) return -100;
    if (block_size < 1 || (block_size & (block_size - 1)) != 0) return -101;
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)o_part) % 16 != 0 || (uintptr_t)ml_part % 8 != 0) return -103;
    for (int i = 0; i < 8; ++i)
        if (strides[i] % 8 != 0) return -103;
    const PlanSizes z = plan_sizes(B, Hq, Hk, 1, 0);
    SharedArgs a;
    a.q = (const char*)q;
    a.kc = (const char*)kc;
    a.vc = (const char*)vc;
    a.block_table = (const int*)block_table;
    a.plan = (const int*)plan;
    a.o_part = (float*)o_part;
    a.ml_part = (float*)ml_part;
    int64_t* const steps[8] = {&a.q_row, &a.q_head, &a.k_page, &a.k_token, &a.k_head, &a.v_page, &a.v_token, &a.v_head};
    for (int i = 0; i < 8; ++i) *steps[i] = strides[i] * 2;
    a.table_row = strides[8];
    a.B = B;
    a.Hq = Hq;
    a.Hk = Hk;
    a.G = Hq / Hk;
    a.pages = pages;
    a.shift = __builtin_ctz(block_size);
    a.slots = z.max_slots;
    a.scale = scale * 1.44269504088896340736f;
    const dim3 grid(z.max_units * Hk), merge(CEIL_DIV(B * Hq, 4)), block(256);
#define LAUNCH(F16, DV, MT)                                                                                     \
    hipLaunchKernelGGL((shared_attn_kernel<F16, DV, MT>), grid, block, 0, (hipStream_t)stream, a)
#define LAUNCH_D(F16, DV)                                                                                       \
    do {                                                                                                        \
        if (z.tile == 16) LAUNCH(F16, DV, 1);                                                                   \
        else if (z.tile == 32) LAUNCH(F16, DV, 2);                                                              \
        else LAUNCH(F16, DV, 4);                                                                                \
        HIP_CHECK_LAUNCH();                                                                                     \
        hipLaunchKernelGGL((shared_combine_kernel<F16, DV>), merge, block, 0, (hipStream_t)stream, a.o_part,    \
                           a.ml_part, a.plan, (char*)out, B, Hq, a.slots);                                      \
        HIP_CHECK_LAUNCH();                                                                                     \
    } while (0)
    if (f16) {
        if (D == 64) LAUNCH_D(true, 64);
        else LAUNCH_D(true, 128);
    } else {
        if (D == 64) LAUNCH_D(false, 64);
        else LAUNCH_D(false, 128);
    }
#undef LAUNCH_D
#undef LAUNCH
    return 0;
}
