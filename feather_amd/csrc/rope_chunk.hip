// Rotary positions of a chunk of new tokens, with the quantisation and the append to the paged cache: every row of a
// ragged batch holds the heads q | k | v of one token; the first rot_dim dims of each q and k head are rotated at the
// token's position, q goes out as packed FP8 words, k and v into the cache slots of the position.
//     (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t),   t = 2 pi * position * freq[pair]
// Pairs are (j, j + rot_dim / 2) (half layout) or (2j, 2j + 1) (interleaved).  freq is in turns per position and in
// 64 bits, and so is the product: far positions make thousands of turns, of which only the fraction counts (a 32-bit
// product around position 10^5 is off by up to 0.001 of a turn).  The fraction is exact to 2^-53 * turns; from there on
// 32 bits do.
//
// A streaming kernel, bound by its bytes: 4 (or 2) in, 1 out per element.  The angles of a token are computed once per
// workgroup and shared by its heads through LDS; the elements are requested before the position is looked up, so the
// two chains overlap.  9 ragged chunks (4505 rows of 48 heads, d = 128, fp32): 138 MB in 37 us, 3.7 TB/s of the 5.1 that
// a copy reaches (27 us), from fp16 83 MB in 32 us; one token for 32 requests (40 heads of 64): 3.7 us, three dependent
// memory round trips.  More units per thread, so that fewer workgroups compute the angles: 2, 3 or 4 of them 41, 37 and
// 39 us, and 4.3, 4.5 and 4.6 us for the single tokens -- not worth it.
#include "rotary.h"

namespace feather {

constexpr int kRcThreads = 256;
constexpr int kRcMaxPairs = 256;      // rot_dim <= 512

struct RopeChunkArgs {
    const void *qkv;
    const int32_t *cu_seqlens, *start_pos, *block_tables;
    const double *freq;
    uint32_t *q_packed, *k_cache, *v_cache;
    int32_t *ctx_after, *status;
    float *rot_f32;
    int64_t row_stride;               // elements between rows of qkv
    int n_seq, total_rows, n_q, n_kv, d, rot, block_size, max_blocks, n_blocks, interleaved, fill;
    float amplitude;
};

// the sequence's answer: how far its positions could be appended, and why not further
__device__ void rope_chunk_status(const RopeChunkArgs &a, int s) {
    const int lane = lane_id();
    const int r0 = min(max(a.cu_seqlens[s], 0), a.total_rows), r1 = max(min(max(a.cu_seqlens[s + 1], 0), a.total_rows), r0);
    const int64_t p0 = a.start_pos[s], p1 = p0 + (r1 - r0), cap = (int64_t)a.max_blocks * a.block_size;
    const int64_t lo = max(p0, (int64_t)0), hi = min(p1, cap);         // positions that have a table entry
    int64_t bad = INT64_MAX;                                            // first position whose entry is not a block
    if (lo < hi)
        for (int64_t e = lo / a.block_size + lane; e <= (hi - 1) / a.block_size; e += kWave)
            if ((unsigned)a.block_tables[(int64_t)s * a.max_blocks + e] >= (unsigned)a.n_blocks) {
                bad = max(e * a.block_size, lo);
                break;
            }
    for (int off = 32; off > 0; off >>= 1) bad = min(bad, (int64_t)__shfl_xor((long long)bad, off, kWave));
    if (lane != 0) return;
    const int64_t reached = p0 < 0 && r1 > r0 ? 0 : min(min(bad, hi), max(p1, (int64_t)0));
    a.ctx_after[s] = (int32_t)(r1 > r0 ? max(min(reached, cap), (int64_t)0) : min(max(p0, (int64_t)0), cap));
    if (a.status) a.status[s] = r1 == r0 ? 0 : ((p0 < 0 || p1 > cap) ? 1 : (bad != INT64_MAX ? 2 : 0));
}

template <bool F16>
__device__ __forceinline__ float4_t rope_load4(const void *p, int64_t at) {
    if constexpr (F16) {
        const half4_t h = __builtin_nontemporal_load(reinterpret_cast<const half4_t *>(static_cast<const _Float16 *>(p) + at));
        return float4_t{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
    } else {
        return __builtin_nontemporal_load(reinterpret_cast<const float4_t *>(static_cast<const float *>(p) + at));
    }
}

// Workgroups [0, n_seq): one wave each answers for a sequence.  The others: `parts` workgroups per token, a unit per
// thread.  A unit is 4 + 4 elements: a pair group of the half layout (elements 4t .. and their partners rot / 2 further
// on), or eight neighbours (interleaved pairs, dims that are not rotated, v).
template <int MODE, bool F16>
__global__ __launch_bounds__(kRcThreads) void rope_chunk_kernel(RopeChunkArgs a, int parts) {
    __shared__ __attribute__((aligned(16))) float cs[2 * kRcMaxPairs];
    if ((int)blockIdx.x < a.n_seq) {
        if (threadIdx.x < kWave) rope_chunk_status(a, blockIdx.x);
        return;
    }
    const int item = blockIdx.x - a.n_seq;
    const int row = item / parts, part = item - row * parts;
    const int heads = a.n_q + 2 * a.n_kv, per_head = a.d / 8, units = heads * per_head;
    const int half = a.rot / 2;
    const int u = part * kRcThreads + (int)threadIdx.x;
    const bool live = u < units;
    const int head = live ? u / per_head : 0, t = live ? u - head * per_head : 0;
    const bool turns = t < a.rot / 8 && head < a.n_q + a.n_kv, split = turns && !a.interleaved;
    const int at_lo = split ? 4 * t : 8 * t, at_hi = split ? half + 4 * t : 8 * t + 4;
    const int64_t from = (int64_t)row * a.row_stride + (int64_t)head * a.d;
    float4_t lo = rope_load4<F16>(a.qkv, from + at_lo), hi = rope_load4<F16>(a.qkv, from + at_hi);
    // ---- the row's sequence: the last one that starts at or before it (64 per step)
    int below = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += kWave) {
        const int s = s0 + lane_id();
        const uint64_t m = __builtin_amdgcn_ballot_w64(s < a.n_seq && a.cu_seqlens[min(s, a.n_seq - 1)] <= row);
        below += __builtin_popcountll(m);
        if (m != ~0ull) break;
    }
    const int seq = __builtin_amdgcn_readfirstlane(below - 1);
    const bool inside = seq >= 0 && row < a.cu_seqlens[max(seq, 0) + 1];
    float *const rot_out = a.rot_f32 ? a.rot_f32 + ((int64_t)row * heads + head) * a.d : nullptr;
    if (!inside) {                                    // a row of no sequence
        if (a.fill && live) {
            if (head < a.n_q) {
                uint32_t *dst = a.q_packed + ((int64_t)row * a.n_q + head) * (a.d / 4);
                dst[at_lo / 4] = 0u;
                dst[at_hi / 4] = 0u;
            }
            if (rot_out) {
                *reinterpret_cast<float4_t *>(rot_out + at_lo) = float4_t{0.f, 0.f, 0.f, 0.f};
                *reinterpret_cast<float4_t *>(rot_out + at_hi) = float4_t{0.f, 0.f, 0.f, 0.f};
            }
        }
        return;
    }
    const int64_t pos = (int64_t)a.start_pos[seq] + (row - max(a.cu_seqlens[seq], 0));
    const bool pos_ok = pos >= 0 && pos < (int64_t)a.max_blocks * a.block_size;
    const int entry = pos_ok ? (int)pos / a.block_size : 0;
    int blk = -1;
    if (pos_ok) blk = a.block_tables[(int64_t)seq * a.max_blocks + entry];
    for (int j = threadIdx.x; j < half; j += kRcThreads) {
        double x = (double)pos * a.freq[j];
        x -= rint(x);                                 // fraction of a turn, [-1/2, 1/2]
        const double k = rint(4.0 * x);
        float s, c;
        sincos_quadrant((float)((x - 0.25 * k) * 6.283185307179586), (int)k, s, c);
        cs[2 * j] = c * a.amplitude;
        cs[2 * j + 1] = s * a.amplitude;
    }
    __syncthreads();
    if (!live) return;
    if (turns) {
        const float4_t p0 = *reinterpret_cast<const float4_t *>(&cs[8 * t]), p1 = *reinterpret_cast<const float4_t *>(&cs[8 * t + 4]);
        const float c[4] = {p0[0], p0[2], p1[0], p1[2]}, s[4] = {p0[1], p0[3], p1[1], p1[3]};
        if (!a.interleaved) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float x = lo[e], y = hi[e];
                lo[e] = x * c[e] - y * s[e];
                hi[e] = y * c[e] + x * s[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float x = lo[2 * e], y = lo[2 * e + 1], z = hi[2 * e], w = hi[2 * e + 1];
                lo[2 * e] = x * c[e] - y * s[e];
                lo[2 * e + 1] = y * c[e] + x * s[e];
                hi[2 * e] = z * c[2 + e] - w * s[2 + e];
                hi[2 * e + 1] = w * c[2 + e] + z * s[2 + e];
            }
        }
    }
    if (rot_out) {                                    // the values the codes are rounded from
        *reinterpret_cast<float4_t *>(rot_out + at_lo) = lo;
        *reinterpret_cast<float4_t *>(rot_out + at_hi) = hi;
    }
    uint32_t *dst;
    if (head < a.n_q) {
        dst = a.q_packed + ((int64_t)row * a.n_q + head) * (a.d / 4);
    } else {
        if ((unsigned)blk >= (unsigned)a.n_blocks) return;
        const bool is_k = head < a.n_q + a.n_kv;
        const int kvh = head - a.n_q - (is_k ? 0 : a.n_kv);
        const int64_t slot = ((int64_t)blk * a.n_kv + kvh) * a.block_size + ((int)pos - entry * a.block_size);
        dst = (is_k ? a.k_cache : a.v_cache) + slot * (a.d / 4);
    }
    const uint32_t wlo = quant4<MODE>(lo[0], lo[1], lo[2], lo[3]), whi = quant4<MODE>(hi[0], hi[1], hi[2], hi[3]);
    if (!split) {                                     // neighbours (8 bytes from a multiple of 8 on: d is one)
        *reinterpret_cast<u32x2 *>(dst + at_lo / 4) = u32x2{wlo, whi};
    } else {
        dst[at_lo / 4] = wlo;
        dst[at_hi / 4] = whi;
    }
}

}  // namespace feather

using namespace feather;

extern "C" int feather_rope_append_chunk(const void *qkv, int src_f16, int64_t row_stride, const void *cu_seqlens,
                                         const void *start_pos, const void *block_tables, const void *freq_f64, float amplitude,
                                         int64_t rot_dim, int layout, void *q_packed, void *k_cache, void *v_cache,
                                         void *ctx_after, void *seq_status, void *rot_f32, int fill, int64_t n_seq,
                                         int64_t total_rows, int64_t n_q_heads, int64_t n_kv_heads, int64_t d, int64_t block_size,
                                         int64_t max_blocks, int64_t n_blocks, int mode, void *stream) {
    const char *me = "feather_rope_append_chunk";
    FEATHER_CHECK(mode == FEATHER_E5M2 || mode == FEATHER_E4M3, FEATHER_EMODE, "%s: mode %d not supported", me, mode);
    FEATHER_CHECK(src_f16 == 0 || src_f16 == 1, FEATHER_EINVAL, "%s: src_f16 must be 0 or 1", me);
    FEATHER_CHECK(fill == 0 || fill == 1, FEATHER_EINVAL, "%s: fill must be 0 or 1", me);
    FEATHER_CHECK(layout == FEATHER_ROPE_HALF || layout == FEATHER_ROPE_INTERLEAVED, FEATHER_EINVAL, "%s: bad layout %d", me, layout);
    FEATHER_CHECK(n_seq >= 0 && total_rows >= 0 && n_q_heads >= 0 && n_kv_heads > 0 && block_size > 0 && max_blocks >= 0 && n_blocks >= 1,
                  FEATHER_EINVAL, "%s: bad shape", me);
    FEATHER_CHECK(d > 0 && d % 8 == 0 && d <= 65536, FEATHER_ESHAPE, "%s: head dim %lld is not a multiple of 8", me, (long long)d);
    FEATHER_CHECK(rot_dim >= 0 && rot_dim % 8 == 0 && rot_dim <= d && rot_dim <= 2 * kRcMaxPairs, FEATHER_ESHAPE,
                  "%s: rot_dim=%lld must be a multiple of 8, at most the head dim and %d", me, (long long)rot_dim, 2 * kRcMaxPairs);
    const int64_t heads = n_q_heads + 2 * n_kv_heads;
    FEATHER_CHECK(heads < (1ll << 20) && heads * d < (1ll << 30), FEATHER_ESHAPE, "%s: too many heads", me);
    FEATHER_CHECK(row_stride >= heads * d && row_stride % 4 == 0, FEATHER_ESHAPE,
                  "%s: row_stride=%lld must be a multiple of 4 and hold %lld elements", me, (long long)row_stride, (long long)(heads * d));
    FEATHER_CHECK(total_rows < (1ll << 30) && n_seq < (1ll << 30) && n_blocks < (1ll << 31) && max_blocks < (1ll << 31) &&
                      block_size < (1ll << 31) && max_blocks * block_size < (1ll << 31),
                  FEATHER_ESHAPE, "%s: shape too large", me);
    if (n_seq == 0 && (total_rows == 0 || !fill)) return FEATHER_OK;
    FEATHER_CHECK(cu_seqlens && (n_seq == 0 || (start_pos && ctx_after && (block_tables || max_blocks == 0))) && (freq_f64 || rot_dim == 0), FEATHER_EINVAL,
                  "%s: null pointer", me);
    FEATHER_CHECK(total_rows == 0 || (qkv && (q_packed || n_q_heads == 0) && k_cache && v_cache), FEATHER_EINVAL, "%s: null pointer", me);
    FEATHER_CHECK(aligned(qkv, src_f16 ? 8 : 16) && aligned(q_packed, 8) && aligned(k_cache, 8) && aligned(v_cache, 8) &&
                      aligned(rot_f32, 16) && aligned(freq_f64, 8) && aligned(cu_seqlens, 4) && aligned(start_pos, 4) &&
                      aligned(block_tables, 4) && aligned(ctx_after, 4) && aligned(seq_status, 4),
                  FEATHER_EINVAL, "%s: misaligned pointer", me);
    const uintptr_t k0 = reinterpret_cast<uintptr_t>(k_cache), v0 = reinterpret_cast<uintptr_t>(v_cache);
    FEATHER_CHECK(total_rows == 0 || (uint64_t)(k0 < v0 ? v0 - k0 : k0 - v0) / ((uint64_t)block_size * d) / (uint64_t)n_kv_heads >= (uint64_t)n_blocks,
                  FEATHER_EINVAL, "%s: k_cache and v_cache overlap", me);
    RopeChunkArgs a;
    a.qkv = qkv; a.cu_seqlens = (const int32_t *)cu_seqlens; a.start_pos = (const int32_t *)start_pos;
    a.block_tables = (const int32_t *)block_tables; a.freq = (const double *)freq_f64; a.q_packed = (uint32_t *)q_packed;
    a.k_cache = (uint32_t *)k_cache; a.v_cache = (uint32_t *)v_cache; a.ctx_after = (int32_t *)ctx_after;
    a.status = (int32_t *)seq_status; a.rot_f32 = (float *)rot_f32; a.row_stride = row_stride; a.n_seq = (int)n_seq;
    a.total_rows = (int)total_rows; a.n_q = (int)n_q_heads; a.n_kv = (int)n_kv_heads; a.d = (int)d; a.rot = (int)rot_dim;
    a.block_size = (int)block_size; a.max_blocks = (int)max_blocks; a.n_blocks = (int)n_blocks;
    a.interleaved = layout == FEATHER_ROPE_INTERLEAVED; a.fill = fill; a.amplitude = amplitude;
    const int64_t units = heads * (d / 8);
    const int64_t parts = (units + kRcThreads - 1) / kRcThreads;
    const int64_t grid = n_seq + total_rows * parts;
    FEATHER_CHECK(grid < (1ll << 31), FEATHER_ESHAPE, "%s: grid too large", me);
#define FEATHER_RC(MM, FF)                                                                                             \
    hipLaunchKernelGGL((rope_chunk_kernel<MM, FF>), dim3((unsigned)grid), dim3(kRcThreads), 0, (hipStream_t)stream, a, (int)parts)
    if (mode == FEATHER_E5M2) { if (src_f16) FEATHER_RC(FEATHER_E5M2, true); else FEATHER_RC(FEATHER_E5M2, false); }
    else { if (src_f16) FEATHER_RC(FEATHER_E4M3, true); else FEATHER_RC(FEATHER_E4M3, false); }
#undef FEATHER_RC
    return check_launch(me);
}
