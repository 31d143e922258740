// Attention over the 8-bit key/value cache (layout: kv_dev.h):
//   o = sum_j w_j v_j / (sum_j w_j + w_sink),  w_j = exp(z_j - max z),  z_j = cap(scale q . k_j),  cap(z) = c tanh(z / c)
// over the tokens j that the row sees (j <= its position, j > its position - window).  A row that sees none gives zeros.
//
// Rows are numbered (token of the sequence, query head of the group) for each key/value head, so that all query heads of
// a group share one pass over the cache.  One pass with the running maximum and sum of the softmax; both products on the
// matrix cores in fp16: codes are exact there, queries are scaled by a power of two per row and probabilities by 2^15, and
// f32 calls split both into the rounded half and the half of what is left (22 bits together), so that nothing of an f32
// query is lost; 16-bit calls take probabilities of 11 bits.  Scores, maxima, sums and outputs are fp32.
//
// The first product is K Q^T and the second V^T P^T: a lane's scores are then of one row, its maximum and sum are scalars
// of the lane, and the probabilities are already the second product's operand.
//   key codes of 16-bit calls as subnormal halves (code + 128) 2^-24, one byte permute per pair: the accumulators start at
//   -128 2^-24 sum q, which takes the 128 out.  The matrix cores align a product by its operands' exponent fields, and a
//   subnormal's is that of 2^-14: ten bits of the sum are lost, 6e-6 of a score (measured on ordinary scores; where scores
//   lie within a few units of each other and are differences of magnitudes of 300, in units of log2, f16 outputs are no
//   more than 1.5e-6 beyond their half step, of values up to 4, against 1e-6 for f32 calls).  Too much for f32
//   key codes of f32 calls, and value codes, as the whole numbers themselves: 1024 + byte less 1152, one more instruction
//   per pair (left in, 128 would make sum p (code + 128) hundreds of times the result)
//   scales of keys multiply the scores; scales of values the probabilities, against a running power of two so that the
//   product is at most 1
#include <atomic>

#include "internal.h"
#include "kv_dev.h"

namespace miqmm {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));

typedef float float16v __attribute__((ext_vector_type(16)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr float MINUS_INF = -__builtin_inff();

// one of the two ways that rows are worked on: tiles of 16 or of 128 rows
struct Share {
    float *part;      // [item][kv head][split]: R x dp numerators, R maxima, R sums (R rows per tile)
    int items;        // tiles at most; 0: none
    int splits;       // workgroups that a tile's cache is cut over
    int least, most;  // sequences of least..most (token, head) rows per key/value head
};

struct AttnLaunch {
    DevKv c;
    DevBatch b;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    int heads, group;
    float scale, softcap;
    int causal, window;
    const float *sinks;
    int shift;  // groups of 16 tokens per scale, as a power of two
    Share few, many;
    Divisor by_group, by_heads, by_few_items, by_few_splits, by_many_splits, by_quads;
};

union Halves {
    half8 v;
    half2v h[4];
    uint32_t u[4];
};

// eight code bytes to subnormal halves
__device__ __forceinline__ half8 widen(uint32_t lo, uint32_t hi) {
    Halves r;
    r.u[0] = __builtin_amdgcn_perm(0u, lo, 0x0c010c00u);
    r.u[1] = __builtin_amdgcn_perm(0u, lo, 0x0c030c02u);
    r.u[2] = __builtin_amdgcn_perm(0u, hi, 0x0c010c00u);
    r.u[3] = __builtin_amdgcn_perm(0u, hi, 0x0c030c02u);
    return r.v;
}

// eight code bytes to the codes as halves: 0x6400 | byte is 1024 + byte
__device__ __forceinline__ half8 widen_centred(uint32_t lo, uint32_t hi) {
    Halves r, c;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u);
    c.u[0] = 0x64806480u;  // 1152
#pragma unroll
    for (int i = 0; i < 4; i++) r.h[i] = r.h[i] - c.h[0];
    return r.v;
}

// x as the fp32 number that it is: rounding a product to half straight from its operands (one instruction) can give
// another half than rounding the fp32 product, and the second half would then be the remainder of the wrong one
__device__ __forceinline__ float settled(float x) {
    asm("" : "+v"(x));
    return x;
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23 & 0xff) - 127; }

// tiles of R rows that a share has in a sequence of n rows
template <int R>
__device__ __forceinline__ int tiles_of(const Share &s, int group, int n) {
    const int rows = n * group;
    return rows >= s.least && rows <= s.most ? (rows + R - 1) / R : 0;
}

// the value of the lane 32 away, exchanged in the registers
__device__ __forceinline__ float other_half(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(threadIdx.x & 32 ? r[0] : r[1]);
}

// a head's sink in units of log2; what overflows there, infinity too, counts as the largest number: all weight is the sink's
__device__ __forceinline__ float sink_of(const AttnLaunch &a, int head) {
    const float x = a.sinks[head] * LOG2E;
    return x > 0x1.fffffep127f ? 0x1.fffffep127f : x;
}

__device__ __forceinline__ void visible(const AttnLaunch &a, int pos, int len, int &lo, int &hi) {
    lo = a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0;  // (pos may be negative, and the window 2^31 - 1)
    hi = a.causal ? min(pos + 1, len) : len;
    hi = max(hi, 0);
}

// cap(z) in units of log2 for N scores x / softcap: c tanh(x), c = softcap log2(e).  Below 0.35 the odd series to x^11 (2e-8
// of the value; the formula with the exponential loses eight bits there), and where no lane of the wave has more, that alone.
template <int N>
__device__ __forceinline__ void cap_scores(float (&x)[N], float c) {
    float big = 0.f, r[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        big = fmaxf(big, fabsf(x[i]));
        const float y = x[i] * x[i];
        float p = __builtin_fmaf(y, c * (-1382.f / 155925.f), c * (62.f / 2835.f));
        p = __builtin_fmaf(y, p, c * (-17.f / 315.f));
        p = __builtin_fmaf(y, p, c * (2.f / 15.f));
        p = __builtin_fmaf(y, p, c * (-1.f / 3.f));
        r[i] = x[i] * __builtin_fmaf(y, p, c);
    }
    if (__ballot(!(big < 0.35f))) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            // (1 - t) / (1 + t), t = exp(-2 |x|)
            const float t = __builtin_amdgcn_exp2f(-2.f * LOG2E * fabsf(x[i]));
            const float y = __builtin_copysignf(c * (1.f - t) * __builtin_amdgcn_rcpf(1.f + t), x[i]);
            if (!(fabsf(x[i]) < 0.35f)) r[i] = y;
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = r[i];
}

// Numbers of a sequence's pages, 64 at a time in the lanes of a register: pages from + step * (0 .. 63).  Neither they nor
// the scales go through scalar loads: those share their counter with LDS reads and come back in any order, so every LDS
// read behind one would wait for the cache's memory.
__device__ __forceinline__ int pages_from(const AttnLaunch &a, int seq, int from, int step) {
    const int page = from + step * (int)(threadIdx.x & 63);
    const int phys = page < a.b.max_pages ? a.b.pages[(int64_t)seq * a.b.max_pages + page] : -1;
    return phys < a.c.n_pages ? phys : -1;  // -1: there is no such page
}

// the scales of a page's four groups of 16 tokens: keys' in lanes 0 .. 3 (of every 8), values' in lanes 4 .. 7
__device__ __forceinline__ float scales_from(const AttnLaunch &a, int phys, int head) {
    const int64_t i = ((int64_t)max(phys, 0) * a.c.kv_heads + head) * a.c.per + ((threadIdx.x & 3) >> a.shift);
    return threadIdx.x & 4 ? a.c.vs[i] : a.c.ks[i];
}

__device__ __forceinline__ float lane_float(float x, int lane) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), lane));
}

// as scalars; NaN where there is no such page, and for a negative scale (the maxima below are taken before the key scales, and
// the values' reference by the largest scale): whoever sees it gets NaN.  Scales of 16 tokens that none of the rows worked on
// together (lo .. hi - 1 for all of them) sees are 0: what stands there is a page's earlier content, and of any size.  Returns
// whether one of the rows sees the lane's 16 tokens.  up: a factor of the lane's scale.
__device__ __forceinline__ bool spread_scales(float &x, float up, int phys, int j0, int lo, int hi, float (&ks)[4], float (&vs)[4]) {
    const int j = j0 + 16 * (threadIdx.x & 3);
    const bool seen = j < hi && j + 16 > lo;
    x = seen ? (phys >= 0 && x >= 0.f ? x * up : __builtin_nanf("")) : 0.f;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        ks[t] = lane_float(x, t);
        vs[t] = lane_float(x, 4 + t);
    }
    return seen;
}

// A barrier for what the waves put into LDS alone: __syncthreads() would also wait for the loads of the page after next.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// x and y in registers of their own, copied here.  A register that a load of the loop's next round writes must not be handed on
// or changed in place: the compiler then copies it at the end of the round, where that waits for the load just issued.  The
// two idle states belong to it: a lane swap must not follow within two instructions of the vector instruction that wrote its
// register (a lane read not within one), and the compiler, which otherwise sees to that, does not look into the block.
// Without them a swap may take what the register held before, which is another value's code.
__device__ __forceinline__ void copy_pair(uint32_t &x, uint32_t &y) {
    uint32_t a, b;
    asm("v_mov_b32 %0, %2\n\tv_mov_b32 %1, %3\n\ts_nop 1" : "=&v"(a), "=v"(b) : "v"(x), "v"(y));
    x = a;
    y = b;
}

// the same for one
__device__ __forceinline__ float copied(float x) {
    float y;
    asm("v_mov_b32 %0, %1\n\ts_nop 1" : "=v"(y) : "v"(x));
    return y;
}

// The order of N LDS reads and their PER matrix instructions each: four reads ahead of the instructions.  Left to itself the
// compiler puts two reads right in front of the two instructions that want them, and a wave waits for LDS every time.
template <int N, int PER>
__device__ __forceinline__ void interleave() {
    __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
    for (int i = 0; i < N - 4; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 4 * PER, 0);
}

// Scales that are no numbers (a poisoned block, a page that there is not) are taken out of a page's work -- masked tokens of
// such a block would turn into NaN -- and make NaN of the sum of a row (lo .. hi - 1) that sees one of the block's tokens.
__device__ __forceinline__ void take_out_nan(float (&ks)[4], float (&vs)[4], int j0, int lo, int hi, float &l) {
    const float all = ks[0] + ks[1] + ks[2] + ks[3] + vs[0] + vs[1] + vs[2] + vs[3];
    if (all - all == 0.f) return;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const float both = ks[t] + vs[t];
        if (both - both == 0.f) continue;
        ks[t] = vs[t] = 0.f;
        if (max(lo, j0 + 16 * t) < min(hi, j0 + 16 * t + 16)) l = __builtin_nanf("");
    }
}

// one past the last page that rows with these bounds see, of those that the table has
__device__ __forceinline__ int last_page(const AttnLaunch &a, int t0, int lo_min, int hi_max) {
    return hi_max > lo_min ? max(t0, min((hi_max - 1) / KV_PAGE + 1, a.b.max_pages)) : t0;
}

// the sum that a row starts with: NaN if it sees tokens behind the table's last page
__device__ __forceinline__ float first_sum(const AttnLaunch &a, int lo, int hi) {
    return hi > lo && (hi - 1) / KV_PAGE >= a.b.max_pages ? __builtin_nanf("") : 0.f;
}

// ---- 16 rows per workgroup: a step of few tokens --------------------------------------------------------------------
// Bound: HBM (the cache is read once; 16 rows are worth 64 flops a byte).  A wave takes whole pages (64 tokens), the four
// waves of a workgroup every fourth one, each with its own running maximum; the workgroup joins them, and where the
// cache is split over workgroups a second kernel joins those.
//
// Measured, f32, 32 query and 8 key/value heads of 128: 64 sequences of up to 8192 tokens 153 us (754 MB, 4.9 TB/s; a copy
// runs at 5.4), bf16 150; one sequence of 4096 tokens 10.7 us (7.3 and the second kernel), of 32768 21.2 (3.2 TB/s), of 131072
// 50.3 (5.3).  Heads of 192 and 256 fill the registers with a page, so that one wave runs per SIMD and nothing hides its page's
// arithmetic: 16 sequences of up to 8192 tokens, 16 and 8 heads of 256, 89 us (393 MB, 4.4 TB/s), one of 32768 42 (3.2).
constexpr int ROWS = 16;

struct RowsLds {
    float o[4][ROWS][64 + 4];
    float m[4][ROWS], l[4][ROWS];
};

// work: the workgroup's number among the share's, heads fastest
template <class T, int NC, bool CAP>
__device__ __forceinline__ void attn_rows(const AttnLaunch &a, RowsLds &lds, int work) {
    constexpr bool HILO = sizeof(T) == 4;                // queries in two halves
    constexpr bool PHILO = !__is_same(T, __bf16);  // probabilities in two halves
    constexpr int DP = 64 * NC;
    using V4 = typename Vec4<T>::type;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int r = lane % 16, g = lane / 16;
    const int rest = divided(work, a.by_heads), head = work - rest * a.c.kv_heads;  // key/value head
    const int split = divided(rest, a.by_few_items), item = rest - split * a.few.items;
    Found at_item;
    if (!find_item(a.b, item, [&](int n, int) { return tiles_of<ROWS>(a.few, a.group, n); }, at_item)) return;
    const int seq = at_item.seq, tile = at_item.local, begin = at_item.begin;
    const int n = at_item.n, len = at_item.len, first = len - n;
    const int rows = n * a.group, row0 = tile * ROWS;
    const bool valid = row0 + r < rows;
    const int my_t = valid ? divided(row0 + r, a.by_group) : 0, my_h = valid ? row0 + r - my_t * a.group : 0;
    int lo, hi;
    visible(a, first + my_t, len, lo, hi);
    int lo_min, lo_max, hi_min, hi_max;  // over the tile's rows: both bounds grow with the row
    visible(a, first + divided(row0, a.by_group), len, lo_min, hi_min);
    visible(a, first + divided(min(row0 + ROWS, rows) - 1, a.by_group), len, lo_max, hi_max);

    // Everything that the rows wait for once is asked for as early as it can be: page numbers, queries, the first page.
    int t0 = lo_min / KV_PAGE, t1 = last_page(a, t0, lo_min, hi_max);
    if (a.few.splits > 1) {
        const int share = divided(t1 - t0 + a.few.splits - 1, a.by_few_splits);
        t0 = t0 + split * share;
        t1 = min(t1, t0 + share);
    }
    int ids = pages_from(a, seq, t0 + wave, 4);
    V4 raw[NC][4];
    {
        const T *p = (const T *)a.q + (int64_t)(begin + my_t) * a.q_stride + (int64_t)(head * a.group + my_h) * a.c.head_dim;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = 64 * c + 16 * g + 4 * i;
                raw[c][i] = V4{};
                if (valid && d < a.c.head_dim) raw[c][i] = *(const V4 *)(p + d);
            }
    }
    uint4 kc[4][NC], vc[4 * NC];
    float sc;
    auto fetch = [&](int phys) {
        const int64_t at = (int64_t)max(phys, 0) * a.c.kv_heads + head;
        sc = scales_from(a, phys, head);
        const uint4 *kp = (const uint4 *)(a.c.k + at * (KV_PAGE * DP)) + lane;
        const uint4 *vp = (const uint4 *)(a.c.v + at * (KV_PAGE * DP)) + lane;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int c = 0; c < NC; c++) kc[t][c] = kp[(t * NC + c) * 64];
#pragma unroll
        for (int d = 0; d < 4 * NC; d++) vc[d] = vp[d * 64];
    };
    int phys = __builtin_amdgcn_readlane(ids, 0);
    if (t0 + wave < t1) fetch(phys);

    // queries: dimensions 64 c + 16 g + 8 i .. + 7 of row r, as the second operand of step (c, i)
    Halves qh[2 * NC], ql[2 * NC];
    float score_scale, minus_bias;
    float key_up = 1.f;  // lanes of key scales: the 2^24 of subnormal codes, where queries are so large that it has no room beside theirs
    {
        float x[NC][16];
        float big = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                x[c][i] = to_f32(raw[c][i / 4][i % 4]);
                big = fmaxf(big, fabsf(x[c][i]));
            }
        big = fmaxf(big, __shfl_xor(big, 16));
        big = fmaxf(big, __shfl_xor(big, 32));
        // the largest magnitude of a row to 2^13 .. 2^14 (for every finite one from 2^-87 on): the halves keep 2^-38 of it
        const int e = min(max(13 - exponent(big), -115), 100);
        const float up = pow2(e);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float y = x[c][i] * up;
                const _Float16 h = (_Float16)y;
                qh[2 * c + i / 8].v[i % 8] = h;
                sum += (float)h;
                if (HILO) {
                    const _Float16 l = (_Float16)(y - (float)h);
                    ql[2 * c + i / 8].v[i % 8] = l;
                    sum += (float)l;
                }
            }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        minus_bias = HILO ? 0.f : sum * (-128.f * 0x1p-24f);
        const bool large = __is_same(T, __bf16) && __ballot(e < -64);  // (f16 ends at 2^16)
        if (large && !(lane & 4)) key_up = 0x1p24f;
        score_scale = a.scale * (HILO || large ? 1.f : 0x1p24f) * pow2(-e) * (CAP ? 1.f / a.softcap : LOG2E);
    }

    float4v acc[4 * NC];
#pragma unroll
    for (int i = 0; i < 4 * NC; i++) acc[i] = float4v{0.f, 0.f, 0.f, 0.f};
    float m = MINUS_INF, l = first_sum(a, lo, hi);
    float ref = 0x1p-100f, unit = 0x1p115f;  // values are accumulated in units of ref * 2^-15 = 1 / unit

    for (int page = t0 + wave, k = 0; page < t1; page += 4, k++) {
        if (k) {
            if (k % 64 == 0) ids = pages_from(a, seq, page, 4);
            phys = __builtin_amdgcn_readlane(ids, k % 64);
            fetch(phys);
        }
        float ks[4], vs[4];
        const int j0 = page * KV_PAGE;
        spread_scales(sc, key_up, phys, j0, lo_min, hi_max, ks, vs);
        take_out_nan(ks, vs, j0, lo, hi, l);
        float z[16];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            float4v s = {minus_bias, minus_bias, minus_bias, minus_bias};
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const half8 k0 = HILO ? widen_centred(kc[t][c].x, kc[t][c].y) : widen(kc[t][c].x, kc[t][c].y);
                const half8 k1 = HILO ? widen_centred(kc[t][c].z, kc[t][c].w) : widen(kc[t][c].z, kc[t][c].w);
                s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[2 * c].v, s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[2 * c + 1].v, s, 0, 0, 0);
                if (HILO) {
                    s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[2 * c].v, s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[2 * c + 1].v, s, 0, 0, 0);
                }
            }
            const float f = score_scale * ks[t];
#pragma unroll
            for (int i = 0; i < 4; i++) z[4 * t + i] = s[i] * f;
        }
        if (CAP) cap_scores(z, a.softcap * LOG2E);
        if (j0 < lo_max || j0 + KV_PAGE > hi_min) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int j = j0 + 16 * (i / 4) + 4 * g + i % 4;
                if (j < lo || j >= hi) z[i] = MINUS_INF;
            }
        }
        float top = z[0];
#pragma unroll
        for (int i = 1; i < 16; i++) top = fmaxf(top, z[i]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float m_new = fmaxf(m, top), base = m_new == MINUS_INF ? 0.f : m_new;
        const float vmax = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
        float keep = __builtin_amdgcn_exp2f(m - base);
        l *= keep;
        if (vmax > ref) {
            const int e = min(exponent(vmax) + 1, 126);
            keep *= ref * pow2(-e);
            ref = pow2(e);
            unit = e >= -100 ? pow2(15 - e) : unit;
        }
        m = m_new;
        if (__ballot(keep != 1.f)) {
#pragma unroll
            for (int i = 0; i < 4 * NC; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][e] *= keep;
        }
        Halves ph[2], pl[2];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float p = __builtin_amdgcn_exp2f(z[i] - base);
            l += p;
            float y = p * (vs[i / 4] * unit);
            if (PHILO) y = settled(y);
            const _Float16 h = (_Float16)y;
            ph[i / 8].v[i % 8] = h;
            if (PHILO) pl[i / 8].v[i % 8] = (_Float16)(y - (float)h);
        }
#pragma unroll
        for (int d = 0; d < 4 * NC; d++) {
            const half8 v0 = widen_centred(vc[d].x, vc[d].y), v1 = widen_centred(vc[d].z, vc[d].w);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0].v, acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[1].v, acc[d], 0, 0, 0);
            if (PHILO) {
                acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0].v, acc[d], 0, 0, 0);
                acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[1].v, acc[d], 0, 0, 0);
            }
        }
    }

    // the four waves' results joined: 64 dimensions at a time through LDS
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) { lds.m[wave][r] = m; lds.l[wave][r] = l; }
    __syncthreads();
    auto joined = [&](int row, float &top, float &base, float &sum) {
        top = fmaxf(fmaxf(lds.m[0][row], lds.m[1][row]), fmaxf(lds.m[2][row], lds.m[3][row]));
        base = top == MINUS_INF ? 0.f : top;
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) sum += __builtin_amdgcn_exp2f(lds.m[w][row] - base) * lds.l[w][row];
    };
    float top, base, sum;
    joined(r, top, base, sum);
    const float weight = __builtin_amdgcn_exp2f(m - base) * (ref * 0x1p-15f);

    const int o_row = tid / 16, o_d = tid % 16 * 4;  // what this thread writes of 64 dimensions
    const bool writes = row0 + o_row < rows;
    const int o_t = writes ? divided(row0 + o_row, a.by_group) : 0, o_h = head * a.group + (writes ? row0 + o_row - o_t * a.group : 0);
    joined(o_row, top, base, sum);
    const int64_t index = ((int64_t)item * a.c.kv_heads + head) * a.few.splits + split;
    float *part = a.few.part + index * (ROWS * (DP + 2));
    float divide = 1.f;
    if (a.few.splits == 1) {
        float total = sum;
        if (a.sinks) {
            const float sink = sink_of(a, o_h), all = fmaxf(base, sink);
            // the sink joins the sum; where it is the largest, everything is measured against it
            divide = __builtin_amdgcn_exp2f(base - all);
            total = sum * divide + __builtin_amdgcn_exp2f(sink - all);
        }
        divide = sum == 0.f ? 0.f : divide / total;
    } else if (writes && tid % 16 == 0) {
        part[ROWS * DP + o_row] = top;
        part[ROWS * DP + ROWS + o_row] = sum;
    }
    T *out = (T *)a.out + (int64_t)(begin + o_t) * a.out_stride + (int64_t)o_h * a.c.head_dim;
#pragma unroll
    for (int c = 0; c < NC; c++) {
        if (c) __syncthreads();
#pragma unroll
        for (int d = 0; d < 4; d++) {
            float4v y = acc[4 * c + d];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] *= weight;
            *(float4v *)&lds.o[wave][r][16 * d + 4 * g] = y;
        }
        __syncthreads();
        float4v y = *(const float4v *)&lds.o[0][o_row][o_d];
#pragma unroll
        for (int w = 1; w < 4; w++) {
            const float4v x = *(const float4v *)&lds.o[w][o_row][o_d];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] += x[e];
        }
        const int d = 64 * c + o_d;
        if (!writes || d >= a.c.head_dim) continue;
        if (a.few.splits == 1) {
            V4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = (T)(sum == 0.f ? 0.f : y[e] * divide);
            *(V4 *)(out + d) = w;
        } else {
            *(float4v *)(part + o_row * DP + d) = y;
        }
    }
}

template <class T, int NC, bool CAP>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnLaunch a) {
    __shared__ RowsLds lds;
    attn_rows<T, NC, CAP>(a, lds, (int)blockIdx.x);
}

// ---- 128 rows per workgroup: prompts ----------------------------------------------------------------------------------
// Bound: the vector ALU beside the matrix cores.  A wave holds 32 rows, the workgroup's four waves share each page of 64
// tokens through LDS: each widens a quarter of the codes, once for all 128 rows, while the matrix instructions of the page
// before run (two buffers; the codes are in registers one page ahead of that).  The exponentials of the softmax and the
// widening take the vector ALU about as long as the products take the matrix cores, and a wave does one after the other: scores,
// softmax and the second product of a page in turn, held apart by a scheduling barrier, and two waves per SIMD (one at heads of
// 192 and 256) hide only part of one behind the other.  The 1024 scores of 32 rows against 32 tokens alone are 16 matrix
// instructions (538 ns) and 128 vector instructions (289 ns), and both together measured 720 ns.  This is how the kernel is
// ordered, no limit of the machine: scores of the next page beside this page's softmax in one wave have not been tried.
//
// Registers: no spills in bf16 at heads of 128; 10 at heads of 64 (see the launch bounds below); f16 at heads of 128 spills 17
// (capped 11), f32 capped there 9; f32 at heads of 256 spills 24 (100 bytes per lane), capped 57 (228 bytes), inside the page loop.
//
// Measured: 2 prompts of 4096 and 2577 tokens, 32 and 8 heads of 128: bf16 244-260 us = 740-786 TFLOP/s (569 us the 16-row
// way, which widens every code for 16 rows at a time), f16 330, f32 372; 2048 rows over 32768 tokens, bf16, 860 TFLOP/s; a large
// library product runs at 1200.  509 rows over 16001 tokens, 16 and 8 heads of 256, capped: f32, whose products are taken
// twice, 354 us = 371 TFLOP/s (742 executed), f16 268, bf16 226.
constexpr int TILE = 128;
constexpr float LAZY = 6.f;

template <class T, int NC, bool CAP>
__device__ __forceinline__ void attn_tile(const AttnLaunch &a, uint8_t *lds, int work) {
    constexpr bool HILO = sizeof(T) == 4;              // queries in two halves
    constexpr bool PHILO = !__is_same(T, __bf16);      // probabilities in two halves
    constexpr int DP = 64 * NC, BYTES = KV_PAGE * DP;  // of a page's keys (and values) of one head
    using V4 = typename Vec4<T>::type;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int r = lane % 32, h = lane / 32;
    // heads fastest: with eight of them every XCD keeps one head's cache in its L2; later tiles (longer ones) first
    const int rest = divided(work, a.by_heads), head = work - rest * a.c.kv_heads;
    const int nth = divided(rest, a.by_many_splits), split = rest - nth * a.many.splits, item = a.many.items - 1 - nth;
    Found at_item;
    if (!find_item(a.b, item, [&](int n, int) { return tiles_of<TILE>(a.many, a.group, n); }, at_item)) return;
    const int seq = at_item.seq, tile = at_item.local, begin = at_item.begin;
    const int n = at_item.n, len = at_item.len, first = len - n;
    const int rows = n * a.group, row0 = tile * TILE, wrow0 = row0 + 32 * wave;
    const bool valid = wrow0 + r < rows;
    const int my_t = valid ? divided(wrow0 + r, a.by_group) : 0, my_h = valid ? wrow0 + r - my_t * a.group : 0;
    int lo, hi, lo_min, lo_max, hi_min, hi_max, w_lo_min, w_lo_max, w_hi_min, w_hi_max;
    visible(a, first + my_t, len, lo, hi);
    visible(a, first + divided(row0, a.by_group), len, lo_min, hi_min);
    visible(a, first + divided(min(row0 + TILE, rows) - 1, a.by_group), len, lo_max, hi_max);
    visible(a, first + divided(min(wrow0, rows - 1), a.by_group), len, w_lo_min, w_hi_min);
    visible(a, first + divided(min(wrow0 + 32, rows) - 1, a.by_group), len, w_lo_max, w_hi_max);

    // Everything that a tile waits for once is asked for as early as it can be: page numbers, queries, the first page.
    int t0 = lo_min / KV_PAGE, t1 = last_page(a, t0, lo_min, hi_max);
    if (a.many.splits > 1) {
        const int share = divided(t1 - t0 + a.many.splits - 1, a.by_many_splits);
        t0 = t0 + split * share;
        t1 = min(t1, t0 + share);
    }
    int ids = pages_from(a, seq, t0, 1);  // this page's, the next one's and the one after's number; scales of the first two
    typename Vec4<T>::type raw[NC][8];
    {
        const T *p = (const T *)a.q + (int64_t)(begin + my_t) * a.q_stride + (int64_t)(head * a.group + my_h) * a.c.head_dim;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int d = 64 * c + 16 * (2 * (i / 4) + h) + 4 * (i % 4);
                raw[c][i] = V4{};
                if (valid && d < a.c.head_dim) raw[c][i] = *(const V4 *)(p + d);
            }
    }
    // A wave's share of a page: codes of 16 tokens (its number) of every 64 dimensions, and NC pieces of 16 dimensions of all
    // tokens; asked for one page ahead, widened and put into LDS in the order the matrix instructions take them.
    uint4 kc[NC], vc[NC];
    float ks[4], vs[4];
    auto fetch = [&](int phys) {
        const int64_t at = (int64_t)max(phys, 0) * a.c.kv_heads + head;
        const uint4 *kp = (const uint4 *)(a.c.k + at * BYTES) + wave * NC * 64 + lane, *vp = (const uint4 *)(a.c.v + at * BYTES) + wave * NC * 64 + lane;
#pragma unroll
        for (int i = 0; i < NC; i++) { kc[i] = kp[i * 64]; vc[i] = vp[i * 64]; }
    };
    auto place = [&](int b) {
        uint8_t *kb = lds + b * 4 * BYTES, *vb = kb + 2 * BYTES;
        const int g = lane / 16, x = lane % 16;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            uint8_t *p = kb + (((wave / 2 * NC + c) * 2 + g / 2) * 2) * 1024 + ((g & 1) * 32 + (wave & 1) * 16 + x) * 16;
            *(half8 *)p = HILO ? widen_centred(kc[c].x, kc[c].y) : widen(kc[c].x, kc[c].y);
            *(half8 *)(p + 1024) = HILO ? widen_centred(kc[c].z, kc[c].w) : widen(kc[c].z, kc[c].w);
        }
#pragma unroll
        for (int i = 0; i < NC; i++) {
            const int dt = wave * NC + i;
            // lanes 32 apart hold tokens 4 g .. and 4 (g + 2) .. of each 16: exchanged, each has both of two sixteens
            uint32_t x0 = vc[i].x, z0 = vc[i].z, y0 = vc[i].y, w0 = vc[i].w;
            copy_pair(x0, z0);
            copy_pair(y0, w0);
            const auto s0 = __builtin_amdgcn_permlane32_swap(x0, z0, false, false);
            const auto s1 = __builtin_amdgcn_permlane32_swap(y0, w0, false, false);
            uint8_t *p = vb + (dt / 2 * 4 + lane / 32 * 2) * 1024 + ((g & 1) * 32 + (dt & 1) * 16 + x) * 16;
            *(half8 *)p = widen_centred(s0[0], s0[1]);
            *(half8 *)(p + 1024) = widen_centred(s1[0], s1[1]);
        }
    };
    int phys = __builtin_amdgcn_readlane(ids, 0), next = __builtin_amdgcn_readlane(ids, 1);
    float sc = scales_from(a, phys, head), next_sc = 0.f;
    fetch(phys);

    // queries: dimensions 64 c + 16 (2 e + h) + 8 i .. + 7 of row r, as the second operand of step (c, e, i)
    Halves qh[NC][2][2], ql[HILO ? NC : 1][2][2];
    float score_scale, minus_bias, key_up = 1.f;  // (see the 16-row kernel)
    {
        float x[NC][2][16];
        float big = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[c][i / 4][4 * (i % 4) + e] = to_f32(raw[c][i][e]);
                    big = fmaxf(big, fabsf(to_f32(raw[c][i][e])));
                }
        big = fmaxf(big, other_half(big));
        const int e = min(max(13 - exponent(big), -115), 100);
        const float up = a.scale < 0.f ? -pow2(e) : pow2(e);  // the scale's sign goes into the queries
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const float y = x[c][i / 16][i % 16] * up;
                const _Float16 z = (_Float16)y;
                qh[c][i / 16][i / 8 % 2].v[i % 8] = z;
                sum += (float)z;
                if (HILO) ql[HILO ? c : 0][i / 16][i / 8 % 2].v[i % 8] = (_Float16)(y - (float)z);
            }
        sum += other_half(sum);
        minus_bias = HILO ? 0.f : sum * (-128.f * 0x1p-24f);
        const bool large = __is_same(T, __bf16) && __ballot(e < -64);
        if (large && !(lane & 4)) key_up = 0x1p24f;
        score_scale = fabsf(a.scale) * (HILO || large ? 1.f : 0x1p24f) * pow2(-e) * (CAP ? 1.f / a.softcap : LOG2E);
    }

    if constexpr (NC == 4) {
        // one wave per SIMD has 256 accumulation registers beside its vector registers: the queries stay there (1024 rows over
        // 16384 tokens, bf16: 731 -> 671 us; at NC = 3 they fit the vector registers)
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                asm("" : "+a"(qh[c][e / 2][e % 2].v));
                if (HILO) asm("" : "+a"(ql[HILO ? c : 0][e / 2][e % 2].v));
            }
    }
    place(0);
    next_sc = scales_from(a, next, head);
    fetch(next);
    float16v acc[2 * NC];
#pragma unroll
    for (int d = 0; d < 2 * NC; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] = 0.f;
    float m = MINUS_INF, l = first_sum(a, lo, hi);
    float ref = 0x1p-100f, unit = 0x1p109f;  // values are accumulated in units of ref * 2^-9 = 1 / unit

    for (int page = t0; page < t1; page++) {
        const int b = (page - t0) & 1;
        lds_barrier();
        const int j0 = page * KV_PAGE;
        const bool seen = spread_scales(sc, key_up, phys, j0, w_lo_min, w_hi_max, ks, vs);
        const bool works = wrow0 < rows && j0 < w_hi_max && j0 + KV_PAGE > w_lo_min;  // else nothing that this wave's rows see
        if (works) {
        take_out_nan(ks, vs, j0, lo, hi, l);
        float f[4], w[4], off[4];  // a score is s * f + off
#pragma unroll
        for (int t = 0; t < 4; t++) {
            f[t] = score_scale * ks[t];
            if (f[t] == 0.f) f[t] = 1e-30f;  // times a masked token's -inf stays -inf; all else is 0 either way
            off[t] = HILO ? 0.f : minus_bias * f[t];
            w[t] = vs[t];
        }
        const half8 *kb = (const half8 *)(lds + b * 4 * BYTES) + lane, *vb = kb + 2 * BYTES / 16;
        // two accumulators in turn: a matrix instruction that continues the one right before it waits for it
        float16v s[2] = {float16v{}, float16v{}};
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const half8 k0 = kb[((c * 2 + e) * 2 + i) * 64], k1 = kb[(((NC + c) * 2 + e) * 2 + i) * 64];
                    s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, qh[c][e][i].v, s[0], 0, 0, 0);
                    s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, qh[c][e][i].v, s[1], 0, 0, 0);
                    if (HILO) {
                        s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, ql[HILO ? c : 0][e][i].v, s[0], 0, 0, 0);
                        s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, ql[HILO ? c : 0][e][i].v, s[1], 0, 0, 0);
                    }
                }
        interleave<8 * NC, HILO ? 2 : 1>();
        if (CAP) {
            float x[32];
#pragma unroll
            for (int i = 0; i < 32; i++) x[i] = __builtin_fmaf(s[i / 16][i % 16], f[i / 8], off[i / 8]);
            cap_scores(x, a.softcap * LOG2E);
#pragma unroll
            for (int i = 0; i < 32; i++) s[i / 16][i % 16] = x[i];
#pragma unroll
            for (int t = 0; t < 4; t++) { f[t] = 1.f; off[t] = 0.f; }
        }
        if (j0 < w_lo_max || j0 + KV_PAGE > w_hi_min) {
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const int j = j0 + 8 * (i / 4) + 4 * h + i % 4;
                if (j < lo || j >= hi) s[i / 16][i % 16] = MINUS_INF;
            }
        }
        float top = MINUS_INF;
#pragma unroll
        for (int t = 0; t < 4; t++) {  // 16 tokens of one scale
            float x = s[t / 2][8 * (t % 2)];
#pragma unroll
            for (int i = 1; i < 8; i++) x = fmaxf(x, s[t / 2][8 * (t % 2) + i]);
            top = fmaxf(top, __builtin_fmaf(x, f[t], off[t]));
        }
        // The row's reference follows its maximum only when that has left it 2^6 behind: among 32 rows one has a new maximum
        // on almost every page, and each time the accumulators are rescaled.  Probabilities are then up to 2^6, and halves
        // hold them times 2^9.
        const float vmax = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
        top = fmaxf(top, other_half(top));
        const bool larger = vmax > ref;  // the same for all lanes
        if (__ballot(top > m + LAZY) || larger) {
            const float m_new = fmaxf(m, top);
            float keep = __builtin_amdgcn_exp2f(m - (m_new == MINUS_INF ? 0.f : m_new));
            l *= keep;
            if (larger) {
                const int e = min(exponent(vmax) + 1, 126);
                keep *= ref * pow2(-e);
                ref = pow2(e);
                unit = e >= -100 ? pow2(9 - e) : unit;
            }
            m = m_new;
#pragma unroll
            for (int d = 0; d < 2 * NC; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) acc[d][i] *= keep;
        }
        const float base = m == MINUS_INF ? 0.f : m;
        Halves ph[4], pl[PHILO ? 4 : 1];
        // 16-bit calls: the value scale goes into the exponent and the sum of the probabilities comes back from the weighted
        // ones -- while no scale is so far below the largest that halves would lose the sum.  Tokens that no row sees have
        // probabilities of 0, whatever their weight; tokens that are seen under a scale of 0 count in the sum with a weight of
        // 0, and a page with such takes the other way: their codes may be anything.  Logarithm and reciprocal of the page's
        // scales are taken once, in the lanes that hold them.
        const float wl = (seen ? sc : ref) * unit;
        if (!HILO && __ballot((lane & 4) && !(wl >= 0x1p-3f)) == 0) {
            const float log_w = __builtin_amdgcn_logf(wl), inv_w = __builtin_amdgcn_rcpf(wl);
            const half2v ones = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const float shift = off[t] - base + lane_float(log_w, 4 + t);
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float y0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t / 2][8 * (t % 2) + i], f[t], shift));
                    const float y1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t / 2][8 * (t % 2) + i + 1], f[t], shift));
                    const half2v x = {(_Float16)y0, (_Float16)y1};
                    ph[t].h[i / 2] = x;
                    if (PHILO) {
                        const half2v rest = {(_Float16)(y0 - (float)x[0]), (_Float16)(y1 - (float)x[1])};
                        pl[PHILO ? t : 0].h[i / 2] = rest;
                        sum += y0 + y1;
                    } else {
                        sum = __builtin_amdgcn_fdot2(x, ones, sum, false);
                    }
                }
                l = __builtin_fmaf(sum, lane_float(inv_w, 4 + t), l);
            }
        } else {
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const float wt = w[t] * unit, shift = off[t] - base;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t / 2][8 * (t % 2) + i], f[t], shift));
                    l += p;
                    float y = p * wt;
                    if (PHILO) y = settled(y);
                    const _Float16 x = (_Float16)y;
                    ph[t].v[i] = x;
                    if (PHILO) pl[PHILO ? t : 0].v[i] = (_Float16)(y - (float)x);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int d = 0; d < 2 * NC; d++) {
                const half8 v = vb[(d * 4 + t) * 64];
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[t].v, acc[d], 0, 0, 0);
                if (PHILO) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[PHILO ? t : 0].v, acc[d], 0, 0, 0);
            }
        interleave<8 * NC, PHILO ? 2 : 1>();
        }
        // The next page into the other buffer, which every wave left before this page's barrier.  Behind the last page this
        // goes on with pages that nobody works on (their number is the table's, or none: then page 0): without a condition
        // the loads go straight into the registers that the next round reads, with one they are waited for here.
        place(b ^ 1);
        sc = copied(next_sc);
        phys = next;
        const int k = page + 2 - t0;
        if (k % 64 == 0) ids = pages_from(a, seq, page + 2, 1);
        next = __builtin_amdgcn_readlane(ids, k % 64);
        next_sc = scales_from(a, next, head);
        fetch(next);
    }

    l += other_half(l);
    if (hi <= lo) l = 0.f;  // sees no token: zeros, also where its own infinities or NaN made the masked scores NaN
    if (!valid) return;
    const int o_h = head * a.group + my_h;
    const float base = m == MINUS_INF ? 0.f : m;
    float weight = ref * 0x1p-9f;
    float *part = a.many.part + (((int64_t)item * a.c.kv_heads + head) * a.many.splits + split) * (TILE * (DP + 2));
    const int in_tile = 32 * wave + r;
    if (a.many.splits == 1) {
        float total = l, scale = 1.f;
        if (a.sinks) {
            const float sink = sink_of(a, o_h), all = fmaxf(base, sink);
            scale = __builtin_amdgcn_exp2f(base - all);
            total = l * scale + __builtin_amdgcn_exp2f(sink - all);
        }
        weight = l == 0.f ? 0.f : weight * (scale / total);
    } else if (h == 0) {
        part[TILE * DP + in_tile] = m;
        part[TILE * DP + TILE + in_tile] = l;
    }
    T *out = (T *)a.out + (int64_t)(begin + my_t) * a.out_stride + (int64_t)o_h * a.c.head_dim;
#pragma unroll
    for (int d = 0; d < 2 * NC; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = 32 * d + 8 * i + 4 * h;
            if (at >= a.c.head_dim) continue;
            float4v y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = l == 0.f ? 0.f : acc[d][4 * i + e] * weight;
            if (a.many.splits == 1) {
                V4 z;
#pragma unroll
                for (int e = 0; e < 4; e++) z[e] = (T)y[e];
                *(V4 *)(out + at) = z;
            } else {
                *(float4v *)(part + in_tile * DP + at) = y;
            }
        }
}

// Prompts, and in the same launch the sequences of few rows beside them: those first, so that single tokens are done while
// the prompts are worked on.
// Waves per SIMD: what the accumulators and queries leave; at heads of 64 three in bf16 pay, with ten spilled registers (2048
// rows over 2048 tokens of 64 heads 81.7 -> 76.5 us), but not where probabilities are in two halves (f16 88.7 -> 94.6, capped
// 110 -> 4448).
template <class T, int NC, bool CAP>
__global__ __launch_bounds__(256, NC == 1 && __is_same(T, __bf16) ? 3 : NC <= 2 ? 2 : 1) void attn_tile_kernel(AttnLaunch a) {
    extern __shared__ __align__(1024) uint8_t lds[];  // two buffers of a page's keys and values as halves
    const int few = a.few.items * a.few.splits * a.c.kv_heads;
    if ((int)blockIdx.x < few) attn_rows<T, NC, CAP>(a, *(RowsLds *)lds, (int)blockIdx.x);
    else attn_tile<T, NC, CAP>(a, lds, (int)blockIdx.x - few);
}

// The splits of a tile joined.  Bound by the latency of its dependent rounds of loads (which sequence, then the partial
// results): a thread takes four dimensions of a row and asks for eight splits' maxima, sums and numerators at a time; where
// that leaves the device empty, G = 8 threads share the splits and join through LDS (a row over 32768 tokens in 128 splits, the whole call: 38.2 us
// with one thread, 24.3 with eight; 512 rows in two splits: 27.6 with one, 55.2 with eight).
template <class T, int R, int G>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnLaunch a) {
    constexpr int W = 256 / G;
    __shared__ float4v lds_y[G > 1 ? G : 1][G > 1 ? W : 1];
    __shared__ float lds_m[G > 1 ? G : 1][G > 1 ? W : 1], lds_l[G > 1 ? G : 1][G > 1 ? W : 1];
    const Share &share = R == ROWS ? a.few : a.many;
    using V4 = typename Vec4<T>::type;
    const int head = blockIdx.y, dp = a.c.dp, quads = a.c.head_dim / 4, w = threadIdx.x % W, g = threadIdx.x / W;
    Found at_item;
    if (!find_item(a.b, (int)blockIdx.x, [&](int n, int) { return tiles_of<R>(share, a.group, n); }, at_item)) return;
    const int tile = at_item.local, begin = at_item.begin, n = at_item.n;
    const int rows = min(R, n * a.group - tile * R);
    const int64_t size = R * (dp + 2);
    const float *part = share.part + ((int64_t)blockIdx.x * a.c.kv_heads + head) * share.splits * size;
    for (int i0 = blockIdx.z * W; i0 < rows * quads; i0 += gridDim.z * W) {
        const int i = i0 + w;
        const bool live = i < rows * quads;
        const int row = live ? divided(i, a.by_quads) : 0, d = live ? (i - row * quads) * 4 : 0;
        const int t = divided(tile * R + row, a.by_group), h = head * a.group + tile * R + row - t * a.group;
        const float sink = a.sinks ? sink_of(a, h) : MINUS_INF;
        float top = MINUS_INF, sum = 0.f;
        float4v y = {0.f, 0.f, 0.f, 0.f};
        // what a further part of the row adds: maximum m, sum l, numerators x; one that saw nothing has no numerators
        auto add = [&](float base, float m, float l, const float4v &x) {
            if (l == 0.f) return;
            const float f = __builtin_amdgcn_exp2f(m - base);
            sum += l * f;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] += x[e] * f;
        };
        if (live) {
            for (int s0 = g; s0 < share.splits; s0 += 8 * G) {
                float m[8], l[8];
                float4v x[8];
#pragma unroll
                for (int s = 0; s < 8; s++) {
                    const float *p = part + min(s0 + G * s, share.splits - 1) * size;
                    m[s] = p[R * dp + row];
                    l[s] = p[R * dp + R + row];
                    x[s] = *(const float4v *)(p + row * dp + d);
                }
                float best = top;
#pragma unroll
                for (int s = 0; s < 8; s++) best = fmaxf(best, m[s]);
                const float base = best == MINUS_INF ? 0.f : best, keep = __builtin_amdgcn_exp2f(top - base);
                top = best;
                sum *= keep;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] *= keep;
#pragma unroll
                for (int s = 0; s < 8; s++)
                    if (s0 + G * s < share.splits) add(base, m[s], l[s], x[s]);
            }
        }
        if constexpr (G > 1) {
            lds_m[g][w] = top;
            lds_l[g][w] = sum;
            lds_y[g][w] = y;
            __syncthreads();
            if (g == 0) {
#pragma unroll
                for (int s = 0; s < G; s++) top = fmaxf(top, lds_m[s][w]);
                sum = 0.f;
                y = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < G; s++) add(top == MINUS_INF ? 0.f : top, lds_m[s][w], lds_l[s][w], lds_y[s][w]);
            }
        }
        if (g == 0 && live) {
            top = top == MINUS_INF ? 0.f : top;
            // the sink joins the sum; where it is the largest, everything is measured against it
            const float all = fmaxf(top, sink), scale = __builtin_amdgcn_exp2f(top - all);
            const float total = sum * scale + (a.sinks ? __builtin_amdgcn_exp2f(sink - all) : 0.f);
            V4 o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = (T)(sum == 0.f ? 0.f : y[e] * scale / total);
            *(V4 *)((T *)a.out + (int64_t)(begin + t) * a.out_stride + (int64_t)h * a.c.head_dim + d) = o;
        }
        if (G > 1) __syncthreads();
    }
}

template <class T, int R>
hipError_t launch_join(const AttnLaunch &a, const Share &share, hipStream_t s) {
    // as many workgroups as the rows that a sequence has on average want; one with more of them goes round
    const int64_t rows = ((int64_t)a.b.n_rows * a.group + a.b.n_seqs - 1) / a.b.n_seqs, values = (rows < R ? rows : R) * (a.c.head_dim / 4);
    const auto grid = [&](int width) { return dim3((unsigned)share.items, (unsigned)a.c.kv_heads, (unsigned)((values + width - 1) / width)); };
    // eight threads for each value where one would not fill the device (two tiles of 8 heads in ten splits: 62.9 us the whole
    // call with eight threads, 55.7 with one)
    if (values * share.items * a.c.kv_heads > 65536) attn_join_kernel<T, R, 1><<<grid(256), 256, 0, s>>>(a);
    else attn_join_kernel<T, R, 8><<<grid(32), 256, 0, s>>>(a);
    return hipGetLastError();
}

template <class T, int NC>
hipError_t launch_one(const AttnLaunch &a, hipStream_t s) {
    const unsigned few = (unsigned)a.few.items * (unsigned)a.few.splits * (unsigned)a.c.kv_heads;
    const unsigned many = (unsigned)a.many.items * (unsigned)a.many.splits * (unsigned)a.c.kv_heads;
    if (!many) {
        if (a.softcap > 0.f) attn_rows_kernel<T, NC, true><<<few, 256, 0, s>>>(a);
        else attn_rows_kernel<T, NC, false><<<few, 256, 0, s>>>(a);
    } else {
        const auto kernel = a.softcap > 0.f ? attn_tile_kernel<T, NC, true> : attn_tile_kernel<T, NC, false>;
        constexpr int lds = 2 * 4 * KV_PAGE * 64 * NC;
        static_assert(lds >= (int)sizeof(RowsLds), "the 16-row way shares the buffers");
        if constexpr (lds > 65536) {
            // More than 64 KiB of dynamic LDS has to be allowed once per device: a bit for each, set by whichever thread comes
            // first (two at once both ask for it, which does no harm); devices without a bit are asked for on every call.
            static std::atomic<uint64_t> allowed[2];
            int dev = 0;
            hipError_t e = hipGetDevice(&dev);
            if (e != hipSuccess) return e;
            const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
            if (!(allowed[a.softcap > 0.f].load(std::memory_order_relaxed) & bit)) {
                e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
                if (e != hipSuccess) return e;
                allowed[a.softcap > 0.f].fetch_or(bit, std::memory_order_relaxed);
            }
        }
        kernel<<<few + many, 256, lds, s>>>(a);
    }
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && few && a.few.splits > 1) e = launch_join<T, ROWS>(a, a.few, s);
    if (e == hipSuccess && many && a.many.splits > 1) e = launch_join<T, TILE>(a, a.many, s);
    return e;
}

template <class T>
hipError_t launch_t(const AttnLaunch &a, hipStream_t s) {
    switch (a.c.dp / 64) {
    case 1: return launch_one<T, 1>(a, s);
    case 2: return launch_one<T, 2>(a, s);
    case 3: return launch_one<T, 3>(a, s);
    default: return launch_one<T, 4>(a, s);
    }
}

// Sequences of at most FEW (token, head) rows per key/value head go the 16-row way, longer ones the 128-row way.
// Measured, 8 key/value heads of 128, f32: 16 sequences of 64 / 96 / 128 rows over up to 4096 tokens 54 / 76 / 86 us the 16-row
// way, 72 / 77 / 82 the other; one sequence over 32768 tokens 44 / 65 / 77 and 49 / 51 / 54.
constexpr int FEW = 64;

// Workgroups that share a tile's cache of `pages` pages, of at most `most` that run at a time for each tile: where a page's
// time (1.2 us at heads of 128, double for f32) over the split's pages, and behind it the joining launch (4 us) and the
// partial results of all rows of the call written and read (`bytes` per split, at 4 TB/s) are least.  32 / 8 heads of 128,
// bf16: 512 rows over their own 512 tokens 21.4 us in one piece, 27.6 in two, 32.3 in four; 64 over 1000 33.6 / 20.1 / 19.5
// in 1 / 4 / 8 pieces; heads of 256, f32: 512 over 512 52.7 / 47.8 / 40.2 in 1 / 2 / 4.
int splits_for(int64_t most, int64_t pages, double page_us, double bytes) {
    int best = 1;
    double least = pages * page_us;
    for (int s = 2; s <= most && s <= pages && s <= 32; s++) {
        const double us = (double)((pages + s - 1) / s) * page_us + 4.0 + s * (2.0 * bytes / 4e6);
        if (us < least) { least = us; best = s; }
    }
    return best;
}

// Both shares with their splits; part is left to the caller.  floats: the partial results of each.  The host knows the width
// of the page table, not the lengths, and plans with it: 512 fresh rows of 32 / 8 heads of 128 are done in one piece under a table
// of 8 pages (21.9 us) and in four under one of 2048 (32.4); a single token over 4096 takes 11.8 and 11.5.
void shares_of(const DevKv &c, const DevBatch &b, const AttnDesc &d, int num_cus, Share &few, Share &many, size_t floats[2]) {
    const int64_t group = d.n_heads / c.kv_heads, all = b.n_rows * group;
    const int64_t active = b.n_seqs < b.n_rows ? b.n_seqs : b.n_rows;
    few = many = Share{nullptr, 0, 1, 1, INT32_MAX};
    floats[0] = floats[1] = 0;
    // what a tile of `rows` rows may see: they are at most that many tokens one after the other
    auto pages_seen = [&](int64_t rows) {
        const int64_t w = d.window > 0 && d.causal ? (d.window + rows) / KV_PAGE + 2 : b.max_pages;
        return w < b.max_pages ? w : (int64_t)b.max_pages;
    };
    // tiles if the rows are spread evenly (items is what there can be at most: for 16 sequences of 128 rows twice as many)
    auto likely = [&](int tile, int64_t seqs) { return seqs * ((all + seqs * tile - 1) / (seqs * tile)); };
    // a row per sequence, or few in all: the 16-row way; one sequence: either; otherwise a launch looks for both
    const bool some_many = all > FEW && b.n_rows > b.n_seqs, some_few = b.n_seqs > 1 || !some_many;
    if (some_few) {
        int64_t items = (all + (ROWS - 1) * active) / ROWS, most = (pages_seen(ROWS) + 3) / 4, want;
        if (some_many) {
            few.most = FEW;
            const int64_t cap = active * ((FEW + ROWS - 1) / ROWS);
            if (items > cap) items = cap;
            // beside prompts: 64 pages per workgroup (16 rounds of its four waves, about 20 us) are done before a prompt is,
            // and up to that length no second launch has to join anything.  The host does not see whether one of the sequences is
            // a prompt, so steps of a few tokens each come here too once they are more than 64 rows: 10 sequences over up to
            // 8192 tokens, 8 / 1 heads of 128, take 14.8 us with one token each, 37.5 with two
            want = (pages_seen(ROWS) + 63) / 64;
        } else {
            // the workgroups that run at a time (three per CU at heads of 64, two at 128; at 192 and 256 one runs, and the second
            // half of the splits a second round), down to a page per wave.  f32, 8
            // heads of 128, two / eight per CU: one sequence of 32768 tokens 21.2 / 24.3 us, of 131072 49.8 / 55.5; 16 of up
            // to 4096 tokens in 3 / 4 / 5 splits 31.1 / 27.0 / 29.9, 32 of up to 8192 in 1 / 2 / 3 80.9 / 83.8 / 88.3
            want = (c.dp <= 64 ? 3ll : 2ll) * num_cus / (likely(ROWS, active) * c.kv_heads);
        }
        few.items = (int)items;
        few.splits = (int)(want < most ? want : most);
        if (few.splits > 256) few.splits = 256;
        if (items * c.kv_heads * few.splits > 65536) few.splits = (int)(65536 / (items * c.kv_heads));  // a GB of partial results
        if (few.splits < 1) few.splits = 1;
        if (few.splits > 1) floats[0] = (size_t)items * c.kv_heads * few.splits * (ROWS * (size_t)(c.dp + 2));
    }
    if (some_many) {
        const int64_t seqs = all / (FEW + 1) < active ? all / (FEW + 1) : active;  // sequences that can be longer than FEW
        many.items = (int)((all + (TILE - 1) * seqs) / TILE);
        if (b.n_seqs > 1) many.least = FEW + 1;
        many.splits = splits_for((c.dp <= 128 ? 2 : 1) * num_cus / (likely(TILE, seqs) * c.kv_heads), pages_seen(TILE),
                                 c.dp / 128.0 * (d.type == T_F32 ? 2.4 : 1.2), 4.0 * (c.dp + 2) * b.n_rows * d.n_heads);
        if (many.splits > 1) floats[1] = (size_t)many.items * c.kv_heads * many.splits * (TILE * (size_t)(c.dp + 2));
    }
}

}  // namespace

size_t attn_workspace_floats(const DevKv &c, const DevBatch &b, const AttnDesc &d, int num_cus) {
    Share few, many;
    size_t floats[2];
    shares_of(c, b, d, num_cus, few, many, floats);
    return floats[0] + floats[1];
}

hipError_t launch_attention(const DevKv &c, const DevBatch &b, const AttnDesc &d, const void *q, int64_t q_stride, void *out,
                            int64_t out_stride, float *workspace, int num_cus, hipStream_t s) {
    AttnLaunch a{c, b, q, out, q_stride, out_stride, d.n_heads, d.n_heads / c.kv_heads, d.scale, d.softcap, d.causal, d.window,
                 d.sinks, c.block == 16 ? 0 : c.block == 32 ? 1 : 2, Share{}, Share{}, {}, {}, {}, {}, {}, {}};
    size_t floats[2];
    shares_of(c, b, d, num_cus, a.few, a.many, floats);
    a.by_group = divisor_of(a.group);
    a.by_heads = divisor_of(c.kv_heads);
    a.by_few_items = divisor_of(a.few.items ? a.few.items : 1);
    a.by_few_splits = divisor_of(a.few.splits);
    a.by_many_splits = divisor_of(a.many.splits);
    a.by_quads = divisor_of(c.head_dim / 4);
    a.few.part = workspace;
    a.many.part = workspace + floats[0];
    if (d.type == T_F32) return launch_t<float>(a, s);
    if (d.type == T_F16) return launch_t<_Float16>(a, s);
    return launch_t<__bf16>(a, s);
}

}  // namespace miqmm
