// Norms of queries and keys for each head and the rotation by position, in one pass over q and k:
//   y = x * (1 / sqrt(mean(x^2) + eps)) * w           over the head_dim values of a head (left out without w)
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t)  for pair i of the n_rot rotated values, t = pos * freq_i
// The pair is (y[i], y[i + n_rot / 2]) or (y[2i], y[2i + 1]); values from n_rot on pass through.
//
// Bound: memory (every value is read and written once); a single token is bound by a launch and two dependent loads.
// Eight values per lane, so that both members of four pairs are in one lane and a head of 128 is 16 lanes: the sum of
// squares is four exchanges inside a row of 16 lanes, and every access is a 16-byte (f32) or 8-byte piece.  The angle is
// formed in turns in fp64 -- pos * freq reaches 1e5 radians, where fp32 holds a few thousandths -- and reduced there, so
// sine and cosine are fp32 functions of a number in -1/2..1/2.  A wave does all its heads of one row with one set of
// sines; rows and heads are divided until about 8192 waves run, then a wave takes more heads of its row.
//
// Measured: 8192 rows of 32 + 8 heads of 128, f32, 336 MB read and written in 68-70 us = 4.8-4.9 TB/s (a copy of 256 MiB
// runs at 5.4), f16 / bf16 41 / 39 us = 4.1-4.3 TB/s (pieces of 8 bytes); one row 4.3-5.1 us a call, the host's time for a launch: the kernel itself takes 3.7-4.0.
#include "internal.h"
#include "kv_dev.h"

namespace miqmm {

namespace {

struct RopeLaunch {
    RopeDesc d;
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_stride, k_stride, q_out_stride, k_out_stride;  // elements between rows
    const int32_t *pos;
    int n, chunks, heads_per_wave;
    Divisor by_chunks;
};

template <int LPH>
__device__ __forceinline__ float head_sum(float s) {  // over the LPH lanes of a head
#pragma unroll
    for (int o = 1; o < LPH; o <<= 1) s += __shfl_xor(s, o);
    return s;
}

// LPH: lanes per head (8, 16, 32: head_dim up to 64, 128, 256); HALVES: pairs are n_rot / 2 apart, otherwise adjacent
template <class T, int LPH, bool HALVES>
__global__ __launch_bounds__(256) void rope_kernel(RopeLaunch a) {
    using V4 = typename Vec4<T>::type;
    constexpr int GROUPS = 64 / LPH;
    const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + threadIdx.x / 64)), lane = threadIdx.x & 63;
    const int row = divided(wave, a.by_chunks), chunk = wave - row * a.chunks;
    if (row >= a.n) return;
    const RopeDesc &d = a.d;
    const int j = lane % LPH, rot_lanes = d.n_rot / 8;
    const bool rotates = j < rot_lanes, live = j < d.head_dim / 8;
    int oa, ob;  // the lane's two groups of four values
    if (!rotates) { oa = d.n_rot + 8 * (j - rot_lanes); ob = oa + 4; }
    else if (HALVES) { oa = 4 * j; ob = d.n_rot / 2 + 4 * j; }
    else { oa = 8 * j; ob = oa + 4; }

    const int all = d.n_heads + d.n_kv_heads;
    int h = chunk * a.heads_per_wave + lane / LPH;
    const int h_end = min(all, (chunk + 1) * a.heads_per_wave);
    const T *q = (const T *)a.q + (int64_t)row * a.q_stride, *k = (const T *)a.k + (int64_t)row * a.k_stride;
    auto load = [&](int head, V4 &x, V4 &y) {
        const T *p = head < d.n_heads ? q + (int64_t)head * d.head_dim : k + (int64_t)(head - d.n_heads) * d.head_dim;
        x = *(const V4 *)(p + oa);
        y = *(const V4 *)(p + ob);
    };
    V4 x0 = {}, x1 = {};
    if (live && h < h_end) load(h, x0, x1);

    float c[4] = {1.f, 1.f, 1.f, 1.f}, s[4] = {0.f, 0.f, 0.f, 0.f};
    if (rotates) {
        const double p = (double)a.pos[row];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double turns = p * (d.freqs[4 * j + i] * 0.15915494309189533577);
            sincospif(2.0f * (float)(turns - rint(turns)), &s[i], &c[i]);
            s[i] *= d.mscale;
            c[i] *= d.mscale;
        }
    }
    float wq[8], wk[8];
    const bool norm_q = d.q_weight != nullptr, norm_k = d.k_weight != nullptr;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        wq[i] = norm_q && live ? d.q_weight[oa + i] : 1.f;
        wq[4 + i] = norm_q && live ? d.q_weight[ob + i] : 1.f;
        wk[i] = norm_k && live ? d.k_weight[oa + i] : 1.f;
        wk[4 + i] = norm_k && live ? d.k_weight[ob + i] : 1.f;
    }
    for (; h < h_end; h += GROUPS) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; i++) { v[i] = to_f32(x0[i]); v[4 + i] = to_f32(x1[i]); }
        if (live && h + GROUPS < h_end) load(h + GROUPS, x0, x1);
        const bool is_q = h < d.n_heads;
        if (is_q ? norm_q : norm_k) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) sum += v[i] * v[i];
            const float scale = 1.0f / sqrtf(head_sum<LPH>(live ? sum : 0.f) / (float)d.head_dim + d.eps);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = v[i] * scale * (is_q ? wq[i] : wk[i]);
        }
        V4 y0, y1;
        if (!rotates) {
#pragma unroll
            for (int i = 0; i < 4; i++) { y0[i] = (T)v[i]; y1[i] = (T)v[4 + i]; }
        } else if (HALVES) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                y0[i] = (T)(v[i] * c[i] - v[4 + i] * s[i]);
                y1[i] = (T)(v[i] * s[i] + v[4 + i] * c[i]);
            }
        } else {
            float r[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                r[2 * i] = v[2 * i] * c[i] - v[2 * i + 1] * s[i];
                r[2 * i + 1] = v[2 * i] * s[i] + v[2 * i + 1] * c[i];
            }
#pragma unroll
            for (int i = 0; i < 4; i++) { y0[i] = (T)r[i]; y1[i] = (T)r[4 + i]; }
        }
        if (live) {
            T *o = is_q ? (T *)a.q_out + (int64_t)row * a.q_out_stride + (int64_t)h * d.head_dim
                        : (T *)a.k_out + (int64_t)row * a.k_out_stride + (int64_t)(h - d.n_heads) * d.head_dim;
            *(V4 *)(o + oa) = y0;
            *(V4 *)(o + ob) = y1;
        }
    }
}

template <class T, int LPH>
hipError_t launch_t(RopeLaunch &a, hipStream_t s) {
    const int groups = 64 / LPH, all = a.d.n_heads + a.d.n_kv_heads, steps = (all + groups - 1) / groups;
    // a wave's heads: one step (64 / LPH heads) each while that leaves at most 8192 waves, more beyond
    int64_t per = ((int64_t)a.n * steps + 8191) / 8192;
    per = per < 1 ? 1 : per > steps ? steps : per;
    a.chunks = (int)((steps + per - 1) / per);
    a.heads_per_wave = (int)per * groups;
    a.by_chunks = divisor_of(a.chunks);
    const int64_t waves = (int64_t)a.n * a.chunks;
    const dim3 grid((unsigned)((waves + 3) / 4));
    if (a.d.halves) rope_kernel<T, LPH, true><<<grid, 256, 0, s>>>(a);
    else rope_kernel<T, LPH, false><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

template <class T>
hipError_t launch_d(RopeLaunch &a, hipStream_t s) {
    if (a.d.head_dim <= 64) return launch_t<T, 8>(a, s);
    if (a.d.head_dim <= 128) return launch_t<T, 16>(a, s);
    return launch_t<T, 32>(a, s);
}

}  // namespace

hipError_t launch_qk_norm_rope(int type, const RopeDesc &d, const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                               const int32_t *pos, int n, void *q_out, int64_t q_out_stride, void *k_out,
                               int64_t k_out_stride, hipStream_t s) {
    RopeLaunch a{d, q, k, q_out, k_out, q_stride, k_stride, q_out_stride, k_out_stride, pos, n, 1, 1, {}};
    if (type == T_F32) return launch_d<float>(a, s);
    if (type == T_F16) return launch_d<_Float16>(a, s);
    return launch_d<__bf16>(a, s);
}

}  // namespace miqmm
