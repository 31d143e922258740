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
//   subnormal's is that of 2^-14: ten bits of the sum are lost, 6e-6 of a score (measured), nothing to 16-bit results but
//   too much for f32
//   key codes of f32 calls, and value codes, as the whole numbers themselves: 1024 + byte less 1152, one more instruction
//   per pair (left in, 128 would make sum p (code + 128) hundreds of times the result)
//   scales of keys multiply the scores; scales of values the probabilities, against a running power of two so that the
//   product is at most 1
#include "internal.h"
#include "kv_dev.h"

namespace miqmm {

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr float MINUS_INF = -__builtin_inff();

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
    float *part;  // [item][kv head][split]: ROWS x dp numerators, ROWS maxima, ROWS sums
    int splits;
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

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exponent(float x) { return (int)(__float_as_uint(x) >> 23 & 0xff) - 127; }

// what the rows of one tile see, and where the tile lies
struct TileRows {
    int begin, n, len, first;  // the sequence: first row, rows, tokens, position of its first row
    int row0, rows;            // first (token, head) row of the tile, and one past the sequence's last
};

__device__ __forceinline__ void visible(const AttnLaunch &a, int pos, int len, int &lo, int &hi) {
    lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    hi = a.causal ? min(pos + 1, len) : len;
    hi = max(hi, 0);
}

// ---- 16 rows per workgroup: a step of few tokens --------------------------------------------------------------------
// Bound: HBM (the cache is read once; 16 rows are worth 64 flops a byte).  A wave takes whole pages (64 tokens), the four
// waves of a workgroup every fourth one, each with its own running maximum; the workgroup joins them, and where the
// cache is split over workgroups a second kernel joins those.
constexpr int ROWS = 16;

template <class T, int NC, bool CAP>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnLaunch a) {
    constexpr bool HILO = sizeof(T) == 4;                // queries in two halves
    constexpr bool PHILO = !__is_same(T, __bf16);  // probabilities in two halves
    constexpr int DP = 64 * NC;
    using V4 = typename Vec4<T>::type;
    __shared__ float part_o[4][ROWS][64 + 4];
    __shared__ float part_m[4][ROWS], part_l[4][ROWS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int r = lane % 16, g = lane / 16;
    const int head = blockIdx.y;  // key/value head
    int seq, tile;
    auto tiles = [&](int s) { int begin; const int n = seq_rows(a.b, s, begin); return (int)(((int64_t)n * a.group + ROWS - 1) / ROWS); };
    if (!find_item(a.b.n_seqs, (int)blockIdx.x, tiles, seq, tile)) return;
    int begin;
    const int n = seq_rows(a.b, seq, begin), len = a.b.kv_len[seq], first = len - n;
    const int rows = n * a.group, row0 = tile * ROWS;
    const bool valid = row0 + r < rows;
    const int my_t = valid ? (row0 + r) / a.group : 0, my_h = valid ? row0 + r - my_t * a.group : 0;
    int lo, hi;
    visible(a, first + my_t, len, lo, hi);
    int lo_min, lo_max, hi_min, hi_max;  // over the tile's rows: both bounds grow with the row
    visible(a, first + row0 / a.group, len, lo_min, hi_min);
    visible(a, first + (min(row0 + ROWS, rows) - 1) / a.group, len, lo_max, hi_max);

    // queries: dimensions 64 c + 16 g + 8 i .. + 7 of row r, as the second operand of step (c, i)
    Halves qh[2 * NC], ql[2 * NC];
    float score_scale, minus_bias;
    {
        float x[NC][16];
        float big = 0.f;
        const T *p = (const T *)a.q + (int64_t)(begin + my_t) * a.q_stride + (int64_t)(head * a.group + my_h) * a.c.head_dim;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = 64 * c + 16 * g + 4 * i;
                V4 y = {};
                if (valid && d < a.c.head_dim) y = *(const V4 *)(p + d);
#pragma unroll
                for (int e = 0; e < 4; e++) { x[c][4 * i + e] = to_f32(y[e]); big = fmaxf(big, fabsf(x[c][4 * i + e])); }
            }
        big = fmaxf(big, __shfl_xor(big, 16));
        big = fmaxf(big, __shfl_xor(big, 32));
        // the largest magnitude of a row to 2^13 .. 2^14: the halves keep 2^-38 of it
        const int e = min(max(13 - exponent(big), -100), 100);
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
        score_scale = a.scale * (HILO ? 1.f : 0x1p24f) * pow2(-e) * (CAP ? 1.f : LOG2E);
    }

    float4v acc[4 * NC];
#pragma unroll
    for (int i = 0; i < 4 * NC; i++) acc[i] = float4v{0.f, 0.f, 0.f, 0.f};
    float m = MINUS_INF, l = 0.f;
    float ref = 0x1p-100f;  // values are accumulated in units of ref * 2^-15

    int t0 = lo_min / KV_PAGE, t1 = hi_max > lo_min ? (hi_max + KV_PAGE - 1) / KV_PAGE : t0;
    if (a.splits > 1) {
        const int share = (t1 - t0 + a.splits - 1) / a.splits;
        t0 = t0 + (int)blockIdx.z * share;
        t1 = min(t1, t0 + share);
    }
    for (int page = t0 + wave; page < t1; page += 4) {
        int64_t phys = page < a.b.max_pages ? a.b.pages[(int64_t)seq * a.b.max_pages + page] : -1;
        const bool bad = phys < 0 || phys >= a.c.n_pages;  // no such page: whoever sees it gets NaN
        if (bad) phys = 0;
        const int64_t at = phys * a.c.kv_heads + head;
        const uint4 *kp = (const uint4 *)(a.c.k + at * (KV_PAGE * DP)) + lane;
        const uint4 *vp = (const uint4 *)(a.c.v + at * (KV_PAGE * DP)) + lane;
        uint4 kc[4][NC], vc[4 * NC];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int c = 0; c < NC; c++) kc[t][c] = kp[(t * NC + c) * 64];
#pragma unroll
        for (int d = 0; d < 4 * NC; d++) vc[d] = vp[d * 64];
        float ks[4], vs[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const int64_t i = at * a.c.per + 16 * t / a.c.block;
            ks[t] = bad ? __builtin_nanf("") : a.c.ks[i];
            vs[t] = bad ? __builtin_nanf("") : a.c.vs[i];
        }
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
            for (int i = 0; i < 4; i++) {
                z[4 * t + i] = s[i] * f;
                if (CAP) z[4 * t + i] = a.softcap * LOG2E * tanhf(z[4 * t + i] / a.softcap);
            }
        }
        const int j0 = page * KV_PAGE;
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
            const float up = pow2(min(exponent(vmax) + 1, 126));
            keep *= ref / up;
            ref = up;
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
            // a masked token counts nothing, whatever its scale is
            const float y = z[i] == MINUS_INF ? 0.f : p * (vs[i / 4] * (0x1p15f / ref));
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
    if (g == 0) { part_m[wave][r] = m; part_l[wave][r] = l; }
    __syncthreads();
    auto joined = [&](int row, float &top, float &base, float &sum) {
        top = fmaxf(fmaxf(part_m[0][row], part_m[1][row]), fmaxf(part_m[2][row], part_m[3][row]));
        base = top == MINUS_INF ? 0.f : top;
        sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) sum += __builtin_amdgcn_exp2f(part_m[w][row] - base) * part_l[w][row];
    };
    float top, base, sum;
    joined(r, top, base, sum);
    const float weight = __builtin_amdgcn_exp2f(m - base) * (ref * 0x1p-15f);

    const int o_row = tid / 16, o_d = tid % 16 * 4;  // what this thread writes of 64 dimensions
    const bool writes = row0 + o_row < rows;
    const int o_t = writes ? (row0 + o_row) / a.group : 0, o_h = head * a.group + (writes ? row0 + o_row - o_t * a.group : 0);
    joined(o_row, top, base, sum);
    const int64_t index = ((int64_t)blockIdx.x * a.c.kv_heads + head) * a.splits + blockIdx.z;
    float *part = a.part + index * (ROWS * (DP + 2));
    float divide = 1.f;
    if (a.splits == 1) {
        float total = sum;
        if (a.sinks) {
            const float sink = a.sinks[o_h] * LOG2E, all = fmaxf(base, sink);
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
            *(float4v *)&part_o[wave][r][16 * d + 4 * g] = y;
        }
        __syncthreads();
        float4v y = *(const float4v *)&part_o[0][o_row][o_d];
#pragma unroll
        for (int w = 1; w < 4; w++) {
            const float4v x = *(const float4v *)&part_o[w][o_row][o_d];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] += x[e];
        }
        const int d = 64 * c + o_d;
        if (!writes || d >= a.c.head_dim) continue;
        if (a.splits == 1) {
            V4 w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = (T)(sum == 0.f ? 0.f : y[e] * divide);
            *(V4 *)(out + d) = w;
        } else {
            *(float4v *)(part + o_row * DP + d) = y;
        }
    }
}

// the splits of a tile joined: a thread takes four dimensions of one row
template <class T>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnLaunch a) {
    using V4 = typename Vec4<T>::type;
    const int head = blockIdx.y, dp = a.c.dp, quads = a.c.head_dim / 4;
    int seq, tile, begin;
    auto tiles = [&](int s) { int x; const int n = seq_rows(a.b, s, x); return (int)(((int64_t)n * a.group + ROWS - 1) / ROWS); };
    if (!find_item(a.b.n_seqs, (int)blockIdx.x, tiles, seq, tile)) return;
    const int n = seq_rows(a.b, seq, begin);
    const int rows = min(ROWS, n * a.group - tile * ROWS);
    const int64_t size = ROWS * (dp + 2);
    const float *part = a.part + ((int64_t)blockIdx.x * a.c.kv_heads + head) * a.splits * size;
    for (int i = threadIdx.x; i < rows * quads; i += 256) {
        const int row = i / quads, d = (i - row * quads) * 4;
        const int t = (tile * ROWS + row) / a.group, h = head * a.group + tile * ROWS + row - t * a.group;
        float top = MINUS_INF;
        for (int s = 0; s < a.splits; s++) top = fmaxf(top, part[s * size + ROWS * dp + row]);
        const float sink = a.sinks ? a.sinks[h] * LOG2E : MINUS_INF;
        top = fmaxf(top, sink);
        const float base = top == MINUS_INF ? 0.f : top;
        float sum = 0.f;
        float4v y = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < a.splits; s++) {
            const float l = part[s * size + ROWS * dp + ROWS + row];
            if (l == 0.f) continue;  // a split that saw nothing
            const float w = __builtin_amdgcn_exp2f(part[s * size + ROWS * dp + row] - base);
            const float4v x = *(const float4v *)(part + s * size + row * dp + d);
            sum += l * w;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] += x[e] * w;
        }
        const float total = sum + (a.sinks ? __builtin_amdgcn_exp2f(sink - base) : 0.f);
        V4 w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = (T)(sum == 0.f ? 0.f : y[e] / total);
        *(V4 *)((T *)a.out + (int64_t)(begin + t) * a.out_stride + (int64_t)h * a.c.head_dim + d) = w;
    }
}

template <class T, int NC>
hipError_t launch_rows(const AttnLaunch &a, dim3 grid, hipStream_t s) {
    if (a.softcap > 0.f) attn_rows_kernel<T, NC, true><<<grid, 256, 0, s>>>(a);
    else attn_rows_kernel<T, NC, false><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

template <class T>
hipError_t launch_t(const AttnLaunch &a, dim3 grid, hipStream_t s) {
    hipError_t e;
    switch (a.c.dp / 64) {
    case 1: e = launch_rows<T, 1>(a, grid, s); break;
    case 2: e = launch_rows<T, 2>(a, grid, s); break;
    case 3: e = launch_rows<T, 3>(a, grid, s); break;
    default: e = launch_rows<T, 4>(a, grid, s); break;
    }
    if (e != hipSuccess || a.splits == 1) return e;
    attn_join_kernel<T><<<dim3(grid.x, grid.y), 256, 0, s>>>(a);
    return hipGetLastError();
}

struct Plan { int64_t items; int splits; };

// Row tiles at most, and workgroups per tile: the cache of a tile is cut until about eight workgroups per CU run (rounds
// of them even out sequences of different lengths), down to one page per wave.
Plan plan_of(const DevKv &c, const DevBatch &b, const AttnDesc &d, int num_cus) {
    const int64_t group = d.n_heads / c.kv_heads;
    const int64_t active = b.n_seqs < b.n_rows ? b.n_seqs : b.n_rows;
    Plan p;
    p.items = (b.n_rows * group + (ROWS - 1) * active) / ROWS;
    int64_t pages = b.max_pages;
    if (d.window > 0) {  // a tile's rows are ROWS / group tokens at most one after the other
        const int64_t w = ((int64_t)d.window + ROWS) / KV_PAGE + 2;
        if (d.causal && w < pages) pages = w;
    }
    const int64_t want = 8ll * num_cus / (p.items * c.kv_heads) + 1, most = (pages + 3) / 4;
    p.splits = (int)(want < most ? want : most);
    if (p.splits < 1) p.splits = 1;
    if (p.splits > 256) p.splits = 256;
    return p;
}

}  // namespace

size_t attn_workspace_floats(const DevKv &c, const DevBatch &b, const AttnDesc &d, int num_cus) {
    const Plan p = plan_of(c, b, d, num_cus);
    return p.splits == 1 ? 0 : (size_t)p.items * c.kv_heads * p.splits * (ROWS * (size_t)(c.dp + 2));
}

hipError_t launch_attention(const DevKv &c, const DevBatch &b, const AttnDesc &d, const void *q, int64_t q_stride, void *out,
                            int64_t out_stride, float *workspace, int num_cus, hipStream_t s) {
    const Plan p = plan_of(c, b, d, num_cus);
    AttnLaunch a{c, b, q, out, q_stride, out_stride, d.n_heads, d.n_heads / c.kv_heads, d.scale, d.softcap, d.causal, d.window,
                 d.sinks, workspace, p.splits};
    const dim3 grid((unsigned)p.items, (unsigned)c.kv_heads, (unsigned)p.splits);
    if (d.type == T_F32) return launch_t<float>(a, grid, s);
    if (d.type == T_F16) return launch_t<_Float16>(a, grid, s);
    return launch_t<__bf16>(a, grid, s);
}

}  // namespace miqmm
