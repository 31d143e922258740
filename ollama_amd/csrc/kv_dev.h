// The 8-bit key/value cache as the kernels see it, and the description of a step's sequences.
//
// Memory of a cache (mi_qmm_kv_create): pages of 64 tokens; per page and key/value head 64 x dp key codes, then in a plane
// of its own 64 x dp value codes, dp = the head dimension rounded up to 64.  A byte holds a code plus 128, so that zero
// extended to 16 bits it is the subnormal half (code + 128) * 2^-24: the attention kernels widen codes with one byte
// permute per pair and no conversion.  Both planes are in the order in which a wave loads matrix-core operands, every load
// of a wave being 1 KiB in a row:
//   key of token t, dimension d:   16-byte pieces [t / 16][d / 64][d % 64 / 16][t % 16], byte d % 16 of the piece
//   value:                         16-byte pieces [d / 16][t % 16 / 4][d % 16],          byte 4 (t / 16) + t % 4
// A lane's key piece is 16 dimensions of one token; its value piece 16 tokens of one dimension, the ones whose scores the
// same lane group holds after the first product, so that the probabilities go into the second without any exchange.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace miqmm {

constexpr int KV_PAGE = 64;

struct DevKv {
    uint8_t *k, *v;         // [n_pages][kv_heads][64 * dp]
    float *ks, *vs;         // [n_pages][kv_heads][64 / block]
    int64_t n_pages;
    int kv_heads, head_dim, dp;
    int block, per;         // tokens per scale, scales per page and head
};

struct DevBatch {
    const int32_t *row_start;  // [n_seqs + 1]
    const int32_t *kv_len;     // [n_seqs]
    const int32_t *pages;      // [n_seqs][max_pages]
    int n_seqs, max_pages;
    int n_rows;
};

// *p as a scalar load where p is the same for the whole wave: nothing that a kernel reads this way is written by it
template <class T>
__device__ __forceinline__ T fixed(const T *p) {
    return *(const __attribute__((address_space(4))) T *)p;
}

// x of the lane that the data-parallel-primitive control names, 0 where there is none or its row of 16 lanes is masked out
template <int CTRL, int ROW_MASK = 0xf>
__device__ __forceinline__ int lane_of(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, ROW_MASK, 0xf, true);
}

// sum over the lanes up to and with the own one: shifts by 1, 2, 4, 8 inside rows of 16, then row totals to the rows after
__device__ __forceinline__ int scan_add(int x) {
    x += lane_of<0x111>(x);
    x += lane_of<0x112>(x);
    x += lane_of<0x114>(x);
    x += lane_of<0x118>(x);
    x += lane_of<0x142, 0xa>(x);
    x += lane_of<0x143, 0xc>(x);
    return x;
}

// Division by a number that the host knows (Granlund and Montgomery 1994): 0 <= x < 2^31, 1 <= d < 2^31.  Three instructions, scalar ones where x is the
// same for a wave; the general division is about forty vector instructions (and as much code to fetch).
struct Divisor {
    uint32_t mul, shift;
};

inline Divisor divisor_of(int64_t d) {
    uint32_t shift = 0;
    while ((int64_t(1) << shift) < d) shift++;
    return Divisor{(uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - (uint64_t)d)) / (uint64_t)d + 1), shift};
}

__device__ __forceinline__ int divided(int x, const Divisor &d) {
    return (int)((__umulhi((uint32_t)x, d.mul) + (uint32_t)x) >> d.shift);
}

// where a work item falls: its sequence, its number there, and the sequence's rows
struct Found {
    int seq, local;
    int begin, n, len;  // first row, rows, tokens
};

// Work items numbered through the sequences, count(n, len) of them in a sequence of n rows and len tokens: where item
// `item` falls.  A row range that is no part of 0..n_rows counts as none.  All lanes of a wave call it together; one round
// of loads per 64 sequences, and while there are more than 256 ahead, one per 256 to pass over them (attention of 2048 single
// tokens over up to 512: 530 -> 441 us).
template <class F>
__device__ __forceinline__ bool find_item(const DevBatch &b, int item, F count, Found &f) {
    const int lane = threadIdx.x & 63;
    int base = 0, s0 = 0;
    auto rows = [&](int begin, int end) { return begin >= 0 && end <= b.n_rows && end > begin ? end - begin : 0; };
    for (; b.n_seqs - s0 > 256; s0 += 256) {
        int begin[4], end[4], len[4], c = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int s = s0 + 64 * i + lane;
            begin[i] = b.row_start[s];
            end[i] = b.row_start[s + 1];
            len[i] = b.kv_len[s];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) c += count(rows(begin[i], end[i]), max(len[i], 0));
        const int total = __builtin_amdgcn_readlane(scan_add(c), 63);
        if (item < base + total) break;
        base += total;
    }
    for (; s0 < b.n_seqs; s0 += 64) {
        const int s = s0 + lane;
        int begin = 0, n = 0, len = 0, c = 0;
        if (s < b.n_seqs) {
            begin = b.row_start[s];
            n = rows(begin, b.row_start[s + 1]);
            len = max(b.kv_len[s], 0);
            c = count(n, len);
        }
        const int incl = scan_add(c);
        const int total = __builtin_amdgcn_readlane(incl, 63);
        if (item < base + total) {
            const int at = __builtin_amdgcn_readfirstlane((int)__builtin_ctzll(__ballot(base + incl > item)));
            f.seq = s0 + at;
            f.local = item - base - __builtin_amdgcn_readlane(incl - c, at);
            f.begin = __builtin_amdgcn_readlane(begin, at);
            f.n = __builtin_amdgcn_readlane(n, at);
            f.len = __builtin_amdgcn_readlane(len, at);
            return true;
        }
        base += total;
    }
    return false;
}

template <class T> struct Vec4 { using type = T __attribute__((ext_vector_type(4))); };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }

}  // namespace miqmm
