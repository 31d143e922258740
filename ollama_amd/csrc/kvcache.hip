// The 8-bit key/value cache: tokens quantized as they are written, and read back (layout: kv_dev.h).
//
// A block of tokens and a head share a scale s = max |x| / 127; codes are x / s rounded to the nearest whole number.  A
// write that goes on in a partly filled block takes s = max(old s, new max / 127) and, where that grew, moves the older
// codes to it: q -> round(q * (old s / s)).  A value that is not finite makes the scale NaN (and every token of the block
// read as NaN) until a write starts the block anew.  All of it is fp32 arithmetic rounded operation by operation, so a
// restatement gives the same bytes.
//
// Bound: memory.  One workgroup per page, head and plane.  Writing, a wave owns the tokens 16 m + 4 g + i (g its number) and
// a lane dp / 64 neighbouring dimensions, so a row of a head is read in one piece, the block's maximum is one exchange
// through LDS, and a lane holds whole 16-byte value pieces; key codes are turned into their pieces through LDS.
//
// Measured, 8 heads of 128, f32: the write of 64 single tokens 4.6 us (7.9 before few tokens had a way of their own), the
// write and read-back of 6091 tokens of four prompts 34-36 us (126 MB, 3.6 TB/s; the read alone runs at 4.9; a workgroup's load,
// maximum and store of its page follow each other with nothing in flight behind them), as bf16 38 (75 MB, 2.0); the read of 65536
// tokens as bf16 82 us (403 MB, 4.9 TB/s; a copy 5.4).  At heads of 256 66 us (251 MB), at heads of up to 64 52 us for half the
// bytes of 128: that instance of the write takes 222 registers, two waves per SIMD, where the one for 128 takes 72.
#include "internal.h"
#include "kv_dev.h"

namespace miqmm {

namespace {

constexpr float PER127 = 0x1.020408p-7f;  // fl(1 / 127)

// pages that the last n of len tokens touch; `table`: those that the page table has
__device__ __forceinline__ int pages_touched(int n, int len, int table) {
    if (n == 0 || len <= 0) return 0;
    return max(0, min((len - 1) / KV_PAGE, table - 1) - max(len - n, 0) / KV_PAGE + 1);
}

// the largest of the wave's values, in lane 63
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    v = max(v, (uint32_t)lane_of<0x111>((int)v));
    v = max(v, (uint32_t)lane_of<0x112>((int)v));
    v = max(v, (uint32_t)lane_of<0x114>((int)v));
    v = max(v, (uint32_t)lane_of<0x118>((int)v));
    v = max(v, (uint32_t)lane_of<0x142, 0xa>((int)v));
    v = max(v, (uint32_t)lane_of<0x143, 0xc>((int)v));
    return v;
}

__device__ __forceinline__ int clamp_code(float r) { return (int)fminf(fmaxf(r, -127.f), 127.f); }

// round(x / s) of the fp32 quotient, for N values.  x * (1 / s) is within 4e-5 of the quotient (127 and two roundings), so
// its nearest whole number is the quotient's unless it lies that close to a half: then, and for scales whose reciprocal is
// not safe, the division itself -- a tenth of the instructions otherwise.
template <int N>
__device__ __forceinline__ void codes_of(const float (&x)[N], float s, int (&q)[N]) {
    const float inv = 1.0f / s;
    float r[N];
    bool sure = s >= 0x1p-100f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float y = x[i] * inv;
        r[i] = rintf(y);
        sure = sure && fabsf(y - r[i]) < 0.4999f;
    }
    if (__ballot(!sure)) {
#pragma unroll
        for (int i = 0; i < N; i++) r[i] = s > 0.f ? rintf(x[i] / s) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < N; i++) q[i] = clamp_code(r[i]) + 128;
}

// One 16-byte piece whose bytes of `mask` hold older codes: moved to the larger scale.
__device__ __forceinline__ void move_piece(uint8_t *p, uint32_t mask, float grown) {
    uint32_t w[4];
    *(uint4 *)w = *(const uint4 *)p;
#pragma unroll
    for (int m = 0; m < 4; m++) {
        uint32_t r = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int byte = (int)(w[m] >> (8 * i) & 0xff);
            const int moved = clamp_code(rintf((float)(byte - 128) * grown)) + 128;
            r |= (uint32_t)(mask >> (4 * m + i) & 1 ? moved : byte) << (8 * i);
        }
        w[m] = r;
    }
    *(uint4 *)p = *(const uint4 *)w;
}

// The codes of tokens lo .. hi - 1 of a page and head, moved by all threads of the workgroup; what is stored to them
// afterwards lands on top.
template <int VEC>
__device__ __forceinline__ void move_codes(uint8_t *codes, bool is_v, int lo, int hi, float grown) {
    for (int i = threadIdx.x; i < 256 * VEC; i += 256) {  // pieces in memory order
        uint32_t mask = 0;
        if (is_v) {
            const int g = i % 64 / 16;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int t = 16 * (j / 4) + 4 * g + j % 4;
                mask |= (uint32_t)(t >= lo && t < hi) << j;
            }
        } else {
            const int t = i / (64 * VEC) * 16 + i % 16;
            mask = t >= lo && t < hi ? 0xffffu : 0u;
        }
        if (mask) move_piece(codes + (int64_t)i * 16, mask, grown);
    }
    __syncthreads();
}

// the block's scale: its older tokens' if there are any and it holds the new largest magnitude (a bit pattern: ordered
// like the numbers, infinity and NaN above all); grown: old / new where the older codes have to move
__device__ __forceinline__ float block_scale(uint32_t big, bool going_on, float old, float &grown, bool &moves) {
    float s = big >= 0x7f800000u ? __builtin_nanf("") : __uint_as_float(big) * PER127;
    if (going_on) {
        if (s <= old || old != old) s = old;
        else if (s > old) { grown = old / s; moves = true; }
    }
    return s;
}

template <class T, int VEC>
__global__ __launch_bounds__(256) void kv_write_kernel(DevKv c, DevBatch b, const T *xk, const T *xv, int64_t k_stride, int64_t v_stride) {
    constexpr int DP = 64 * VEC, PITCH = DP + 16;
    __shared__ uint32_t largest[4][4];                       // [wave][16 tokens]
    __shared__ __align__(16) uint8_t tile[KV_PAGE * PITCH];  // key codes by token
    const int tid = threadIdx.x, lane = tid & 63, g = __builtin_amdgcn_readfirstlane(tid / 64);
    const int head = blockIdx.y;
    const bool is_v = blockIdx.z;
    Found f;
    if (!find_item(b, (int)blockIdx.x, [&](int n, int len) { return pages_touched(n, len, b.max_pages); }, f)) return;
    const int len = f.len, first = len - f.n;
    const int pi = max(first, 0) / KV_PAGE + f.local;
    const int phys = fixed(b.pages + (int64_t)f.seq * b.max_pages + pi);
    const bool there = phys >= 0 && phys < c.n_pages;
    const int t_lo = max(first - pi * KV_PAGE, 0), t_hi = min(len - pi * KV_PAGE, KV_PAGE);  // the page's new tokens
    const T *src = is_v ? xv : xk;
    const int64_t stride = is_v ? v_stride : k_stride;
    const int64_t row0 = (int64_t)f.begin + (pi * KV_PAGE - first);  // row of the page's token 0 (may lie before the sequence)
    const bool live = lane * VEC < c.head_dim;
    const int64_t at = (int64_t)(there ? phys : 0) * c.kv_heads + head;
    float *scales = (is_v ? c.vs : c.ks) + at * c.per;
    uint8_t *codes = (is_v ? c.v : c.k) + at * (KV_PAGE * DP);
    const int going_on = t_lo % c.block ? t_lo / c.block : -1;  // the block that holds older tokens
    float grown = 0.f;
    bool moves = false;

    // A step of few tokens: a wave each, its codes stored byte by byte.  The page's way below would be 20 KiB of code to
    // fetch for one token.
    if (t_hi - t_lo <= 4) {
        const int t = t_lo + g;
        float x[VEC];
        uint32_t big = 0;
#pragma unroll
        for (int v = 0; v < VEC; v++) x[v] = 0.f;
        if (t < t_hi) {
            const T *p = src + (row0 + t) * stride + (int64_t)head * c.head_dim + lane * VEC;
#pragma unroll
            for (int v = 0; v < VEC; v++) {
                if (live && lane * VEC + v < c.head_dim) x[v] = to_f32(p[v]);
                big = max(big, __float_as_uint(x[v]) & 0x7fffffffu);
            }
        }
        if (!there) return;
        const float old = going_on >= 0 ? scales[going_on] : 0.f;
        big = wave_umax(big);
        if (lane == 63) largest[0][g] = big;
        __syncthreads();
        const int block0 = t_lo / c.block, mine = min(t, t_hi - 1) / c.block;  // few tokens lie in two blocks at most
        uint32_t mx0 = 0, mx1 = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (t_lo + i >= t_hi) continue;
            if ((t_lo + i) / c.block == block0) mx0 = max(mx0, largest[0][i]);
            else mx1 = max(mx1, largest[0][i]);
        }
        const float s0 = block_scale(mx0, going_on >= 0, old, grown, moves), s1 = block_scale(mx1, false, 0.f, grown, moves);
        if (moves) move_codes<VEC>(codes, is_v, going_on * c.block, t_lo, grown);
        if (t >= t_hi) return;
        const float s = mine == block0 ? s0 : s1;
        if (lane == 0) scales[mine] = s;  // the tokens of a block write the same
        int q[VEC];
        codes_of(x, s, q);
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            const int d = lane * VEC + v;
            if (d >= c.head_dim) continue;
            const int place = is_v ? ((d / 16 * 4 + t % 16 / 4) * 16 + d % 16) * 16 + t / 16 * 4 + t % 4
                                   : (((t / 16 * VEC + d / 64) * 4 + d % 64 / 16) * 16 + t % 16) * 16 + d % 16;
            codes[place] = (uint8_t)q[v];
        }
        return;
    }

    // the values first: they are asked for before it is known which page they go to
    float x[16][VEC];
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const int t = 16 * (j / 4) + 4 * g + j % 4;
#pragma unroll
        for (int v = 0; v < VEC; v++) x[j][v] = 0.f;
        if (t >= t_lo && t < t_hi) {
            const T *p = src + (row0 + t) * stride + (int64_t)head * c.head_dim + lane * VEC;
#pragma unroll
            for (int v = 0; v < VEC; v++)
                if (live && lane * VEC + v < c.head_dim) x[j][v] = to_f32(p[v]);
        }
    }
    if (!there) return;
    const float old = going_on >= 0 ? scales[going_on] : 0.f;
#pragma unroll
    for (int m = 0; m < 4; m++) {
        uint32_t big = 0;
#pragma unroll
        for (int j = 4 * m; j < 4 * m + 4; j++)
#pragma unroll
            for (int v = 0; v < VEC; v++) big = max(big, __float_as_uint(x[j][v]) & 0x7fffffffu);
        big = wave_umax(big);
        if (lane == 63) largest[g][m] = big;
    }
    __syncthreads();
    float s[4];  // scale of the block that 16 tokens belong to
    {
        uint32_t mx[4];
#pragma unroll
        for (int m = 0; m < 4; m++) mx[m] = max(max(largest[0][m], largest[1][m]), max(largest[2][m], largest[3][m]));
        if (c.block >= 32) { mx[0] = mx[1] = max(mx[0], mx[1]); mx[2] = mx[3] = max(mx[2], mx[3]); }
        if (c.block >= 64) { mx[0] = mx[1] = mx[2] = mx[3] = max(mx[0], mx[2]); }
#pragma unroll
        for (int m = 0; m < 4; m++) s[m] = block_scale(mx[m], 16 * m / c.block == going_on, old, grown, moves);
    }
    if (moves) move_codes<VEC>(codes, is_v, going_on * c.block, t_lo, grown);
    if (tid < c.per && tid >= t_lo / c.block && tid <= (t_hi - 1) / c.block) {
        const int m = tid * c.block / 16;
        scales[tid] = m < 2 ? (m == 0 ? s[0] : s[1]) : (m == 2 ? s[2] : s[3]);
    }
    int q[16][VEC];
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const int t = 16 * (j / 4) + 4 * g + j % 4;
        if (t >= t_lo && t < t_hi) codes_of(x[j], s[j / 4], q[j]);
    }
    if (is_v) {
        bool all = true;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int t = 16 * (j / 4) + 4 * g + j % 4;
            all &= t >= t_lo && t < t_hi;
        }
#pragma unroll
        for (int v = 0; v < VEC; v++) {
            const int d = lane * VEC + v;
            if (d >= c.head_dim) continue;
            uint8_t *piece = codes + (((d / 16) * 4 + g) * 16 + d % 16) * 16;
            if (all) {
                uint32_t w[4];
#pragma unroll
                for (int m = 0; m < 4; m++)
                    w[m] = (uint32_t)q[4 * m][v] | (uint32_t)q[4 * m + 1][v] << 8 | (uint32_t)q[4 * m + 2][v] << 16 | (uint32_t)q[4 * m + 3][v] << 24;
                *(uint4 *)piece = *(const uint4 *)w;
            } else {
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const int t = 16 * (j / 4) + 4 * g + j % 4;
                    if (t >= t_lo && t < t_hi) piece[j] = (uint8_t)q[j][v];
                }
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const int t = 16 * (j / 4) + 4 * g + j % 4;
        if (t >= t_lo && t < t_hi) {
#pragma unroll
            for (int v = 0; v < VEC; v++) tile[t * PITCH + lane * VEC + v] = (uint8_t)q[j][v];
        }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; e++) {  // pieces (64 dimensions e, 16 of them, token), token fastest
        const int t = tid & 63, p = tid / 64;
        if (t >= t_lo && t < t_hi)
            *(uint4 *)(codes + (((t / 16 * VEC + e) * 4 + p) * 16 + t % 16) * 16) = *(const uint4 *)(tile + t * PITCH + e * 64 + p * 16);
    }
}

template <class T, int VEC>
__global__ __launch_bounds__(256) void kv_read_kernel(DevKv c, DevBatch b, T *yk, T *yv, int64_t k_stride, int64_t v_stride) {
    constexpr int DP = 64 * VEC, PITCH = DP + 16;
    constexpr int OUT = 16 / (int)sizeof(T);  // values of a 16-byte store
    __shared__ __align__(16) uint8_t tile[KV_PAGE * PITCH];  // codes by token
    const int tid = threadIdx.x, head = blockIdx.y;
    const bool is_v = blockIdx.z;
    Found f;
    if (!find_item(b, (int)blockIdx.x, [&](int n, int len) { return pages_touched(n, len, INT32_MAX); }, f)) return;
    const int len = f.len, first = len - f.n;
    const int pi = max(first, 0) / KV_PAGE + f.local;
    int phys = pi < b.max_pages ? fixed(b.pages + (int64_t)f.seq * b.max_pages + pi) : -1;
    const bool bad = phys < 0 || phys >= c.n_pages;  // such a page's tokens read as NaN
    if (bad) phys = 0;
    const int t_lo = max(first - pi * KV_PAGE, 0), t_hi = min(len - pi * KV_PAGE, KV_PAGE);
    T *dst = is_v ? yv : yk;
    const int64_t stride = is_v ? v_stride : k_stride;
    const int64_t row0 = (int64_t)f.begin + (pi * KV_PAGE - first);
    const int64_t at = (int64_t)phys * c.kv_heads + head;
    const float *scales = (is_v ? c.vs : c.ks) + at * c.per;
    const uint8_t *codes = (is_v ? c.v : c.k) + at * (KV_PAGE * DP);
    float s[4];
#pragma unroll
    for (int m = 0; m < 4; m++) s[m] = bad ? __builtin_nanf("") : scales[16 * m / c.block];
#pragma unroll
    for (int e = 0; e < VEC; e++) {
        const int i = e * 256 + tid;  // piece in memory order
        const uint4 w = *(const uint4 *)(codes + (int64_t)i * 16);
        if (!is_v) {
            const int t = i / (64 * VEC) * 16 + i % 16, d = i % (64 * VEC) / 64 * 64 + i % 64 / 16 * 16;
            *(uint4 *)(tile + t * PITCH + d) = w;
        } else {
            const int d = i / 64 * 16 + i % 16, g = i % 64 / 16;
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
            // four lanes hold four tokens of four dimensions: turned over, each has four dimensions of one token
            const int u = tid & 3;
#pragma unroll
            for (int m = 0; m < 4; m++) {
                const uint32_t b1 = (uint32_t)lane_of<0xB1>((int)ws[m]);  // of lane ^ 1
                const uint32_t a = u & 1 ? __builtin_amdgcn_perm(ws[m], b1, 0x07030501u) : __builtin_amdgcn_perm(b1, ws[m], 0x06020400u);
                const uint32_t b2 = (uint32_t)lane_of<0x4E>((int)a);      // of lane ^ 2
                const uint32_t r = u & 2 ? __builtin_amdgcn_perm(a, b2, 0x07060302u) : __builtin_amdgcn_perm(b2, a, 0x05040100u);
                *(uint32_t *)(tile + (16 * m + 4 * g + u) * PITCH + d - u) = r;
            }
        }
    }
    __syncthreads();
    const int per_row = c.head_dim / OUT;
    const int step_t = 256 / per_row, step_c = 256 % per_row;
    int t = t_lo + tid / per_row, p = tid % per_row;
    while (t < t_hi) {
        const float sc = t < 32 ? (t < 16 ? s[0] : s[1]) : (t < 48 ? s[2] : s[3]);
        const uint32_t *w = (const uint32_t *)(tile + t * PITCH + p * OUT);
        T out[OUT] __attribute__((aligned(16)));
#pragma unroll
        for (int i = 0; i < OUT; i++) out[i] = (T)((float)((int)(w[i / 4] >> (8 * (i % 4)) & 0xff) - 128) * sc);
        *(uint4 *)(dst + (row0 + t) * stride + (int64_t)head * c.head_dim + p * OUT) = *(const uint4 *)out;
        t += step_t;
        p += step_c;
        if (p >= per_row) { p -= per_row; t++; }
    }
}

template <class T>
hipError_t write_t(const DevKv &c, const DevBatch &b, const void *k, const void *v, int64_t ks, int64_t vs, dim3 grid, hipStream_t s) {
    switch (c.dp / 64) {
    case 1: kv_write_kernel<T, 1><<<grid, 256, 0, s>>>(c, b, (const T *)k, (const T *)v, ks, vs); break;
    case 2: kv_write_kernel<T, 2><<<grid, 256, 0, s>>>(c, b, (const T *)k, (const T *)v, ks, vs); break;
    case 3: kv_write_kernel<T, 3><<<grid, 256, 0, s>>>(c, b, (const T *)k, (const T *)v, ks, vs); break;
    default: kv_write_kernel<T, 4><<<grid, 256, 0, s>>>(c, b, (const T *)k, (const T *)v, ks, vs); break;
    }
    return hipGetLastError();
}

template <class T>
hipError_t read_t(const DevKv &c, const DevBatch &b, void *k, void *v, int64_t ks, int64_t vs, dim3 grid, hipStream_t s) {
    switch (c.dp / 64) {
    case 1: kv_read_kernel<T, 1><<<grid, 256, 0, s>>>(c, b, (T *)k, (T *)v, ks, vs); break;
    case 2: kv_read_kernel<T, 2><<<grid, 256, 0, s>>>(c, b, (T *)k, (T *)v, ks, vs); break;
    case 3: kv_read_kernel<T, 3><<<grid, 256, 0, s>>>(c, b, (T *)k, (T *)v, ks, vs); break;
    default: kv_read_kernel<T, 4><<<grid, 256, 0, s>>>(c, b, (T *)k, (T *)v, ks, vs); break;
    }
    return hipGetLastError();
}

// at most this many (sequence, page) pairs: every one holds a row, and a sequence's rows touch ceil(n / 64) + 1 pages at most
unsigned page_items(const DevBatch &b) {
    const int64_t most = b.n_rows / KV_PAGE + 2 * (int64_t)b.n_seqs;
    return (unsigned)(most < b.n_rows ? most : b.n_rows);
}

}  // namespace

hipError_t launch_kv_write(const DevKv &c, const DevBatch &b, int type, const void *k, const void *v, int64_t k_stride,
                           int64_t v_stride, hipStream_t s) {
    const dim3 grid(page_items(b), (unsigned)c.kv_heads, 2);
    if (type == T_F32) return write_t<float>(c, b, k, v, k_stride, v_stride, grid, s);
    if (type == T_F16) return write_t<_Float16>(c, b, k, v, k_stride, v_stride, grid, s);
    return write_t<__bf16>(c, b, k, v, k_stride, v_stride, grid, s);
}

hipError_t launch_kv_read(const DevKv &c, const DevBatch &b, int type, void *k, void *v, int64_t k_stride, int64_t v_stride,
                          hipStream_t s) {
    const dim3 grid(page_items(b), (unsigned)c.kv_heads, 2);
    if (type == T_F32) return read_t<float>(c, b, k, v, k_stride, v_stride, grid, s);
    if (type == T_F16) return read_t<_Float16>(c, b, k, v, k_stride, v_stride, grid, s);
    return read_t<__bf16>(c, b, k, v, k_stride, v_stride, grid, s);
}

}  // namespace miqmm
