// Attention of a chunk of new tokens over the paged FP8 cache: every sequence of a batch brings a run of new rows
// (one drafted token or thousands of prompt tokens, cu_seqlens) whose K and V are the last ones of its cached context,
//     O[r, h] = sum_k P[k] V[k] / sum_k P[k],   P[k] = exp(scale * Q[r, h] . K[k])   over the visible keys k:
//     causal: k <= ctx - n + r for row r of n (the rows are the last n of the ctx cached tokens); otherwise k < ctx
//     (an encoder's states, whose number has nothing to do with n).
//
// Columns.  The query heads that share a KV head (grouped-query attention) read the same keys, so the unit of work is
// a COLUMN: column c of a (sequence, KV head) pair is row c / group, query head kvh * group + c % group.  A tile of
// columns is one workgroup's work whatever the mix of rows and heads; K and V are then read once for the whole group.
//
// Matrix cores.  S^T[key, col] = K Q^T and O^T[dim, col] += V^T P^T, as in the prefill kernel (attention.hip): a lane
// keeps one column, the accumulator layout of S^T is the B-operand layout of the second product when V^T is written
// to LDS in a permuted key order, so P stays in registers.  E5M2 K and Q go to the matrix core as bf8 bytes.
//
// Numerics.  fp16 x fp16 (or bf8 x bf8) products summed in fp32, softmax statistics in fp32.  P is rounded to fp16
// (nearest even) before it multiplies V, as in the other attention kernels: the second product then runs at the fp16
// rate, and the error (at most 2^-11 of each P) is of the size of the fp16 result's own rounding.  The denominator sums
// the rounded P.  P is scaled so that the largest one is 2^8 or more (kShift): then a P of 2^-22 of the largest is still a
// normal half, one below it is off by at most 2^-33 of the largest, and none above 2^-33 vanishes.  (With the largest at
// 1, many equal keys at 2^-25 of one dominating key were lost altogether.)
//
// Kernels.  Many columns: K and V tiles through LDS, shared by a workgroup's waves -- chunk_attn32_body (d = 64, 128) on
// the 32x32 matrix instructions, chunk_attn_body (d = 256, 512) on the 16x16 ones.  Few columns: chunk_narrow_body, where
// the bytes of the cache bound the call.  A batch that has both runs both, in one grid where the workgroups are alike.
// Key ranges share a column out over more workgroups, chunk_merge_kernel adds them up.
//
// Measured (a chunk of 2048 rows whose last key is 8192, causal; products and sums of the visible keys, merge included):
//     d = 64, 32 heads on 4    E5M2 137 + 11 us, 810 TFLOP/s    E4M3 164 + 11 us, 690 TFLOP/s
//     d = 128, 32 on 8         E5M2 238 us, 1010 TFLOP/s        E4M3 321 us, 750 TFLOP/s
//     d = 256, 8 on 8          E5M2 197 + 14 us, 570 TFLOP/s    E4M3 211 + 14 us, 530 TFLOP/s
//     d = 512, 8 on 8          E5M2 414 + 26 us, 550 TFLOP/s    E4M3 545 + 25 us, 420 TFLOP/s
// (a plain fp16 product of 8192^3 on the same card: 1168).  Bound: vector issue beside the matrix cores up to d = 128 (the
// exponentials, the decode); LDS reads from d = 256 on (16 columns per wave read every K and V tile once per wave: twice
// the time of the products), which more columns per wave would halve if the accumulators left registers for them.
#include <cmath>
#include <type_traits>

#include "common.h"

namespace feather {

typedef float float2p_t __attribute__((ext_vector_type(2)));

struct ChunkArgs {
    const uint32_t *q, *k_cache, *v_cache;
    const int32_t *block_tables, *cu_seqlens, *ctx_lens;
    void *out;
    float *part;            // partial results of the LDS kernel's key ranges (z_wide > 1), then the (maximum, sum) pairs
    int n_seq, total_rows, n_q_heads, n_kv_heads, group, block_size, max_blocks;
    uint32_t max_blk;       // last block of the cache: an entry outside the cache is read as this one
    uint32_t div_mul, group_mul, kv_mul, head_mul;   // x / size = umulhi(2 x, mul) >> shift for 0 <= x < 2^31 (block_size, group, n_kv_heads, n_q_heads)
    int div_shift, group_shift, kv_shift, head_shift;
    int causal, out_kind, fill;
    int z_wide, z_narrow;             // most key ranges of a tile in either kernel
    float per_group;                  // KV heads over the workgroups of the narrow kernel that the chip holds at once
    int narrow_tiles;                 // tiles of a sequence in the narrow kernel, if its rows are bounded as the caller says
    int narrow_rows;                  // beside the LDS kernel: rows a sequence of the narrow one can have (0: it runs alone)
    float *part_narrow;               // its partial results, then the (maximum, sum) pairs, then the keys per range
    int col_split;                    // sequences of more columns than this take the LDS kernel, the others the narrow one
    float scale_log2e;
    float shift_raw, raise_raw;       // kShift and kShift + kLazy as differences of raw scores
};

// What a tile of `qt` columns works on: its sequence, and how many keys its columns can see.
struct ChunkTile {
    int seq, row0, rows;    // first row of the sequence and its number of rows
    int col0, cols;         // first column of the tile; columns of the whole sequence (of one KV head)
    int ctx, p0;            // cached tokens; position of the sequence's row 0 (negative: rows before the cache's first key)
    int keys;               // keys [0, keys) are visible to some column of the tile
};

// Tile slots: sequence s owns slots [cu[s] * group / qt + s, ...).  Each sequence has at least as many slots as it
// needs (floor(a + b) - floor(a) + 1 >= ceil(b)), and the number of all slots follows from total_rows and n_seq, so
// the grid needs no lengths on the host.  The sequence of a slot is the last one whose first slot is not above it:
// 64 sequences are looked at per step, one memory round trip each.
__device__ __forceinline__ int chunk_clamp_row(int r, int total) { return min(max(r, 0), total); }

__device__ __forceinline__ int chunk_row_of(const ChunkArgs &a, int col) { return (int)(__umulhi(2u * (uint32_t)col, a.group_mul) >> a.group_shift); }

// sequence s, its tile from column col0 on
__device__ __forceinline__ void chunk_tile_at(const ChunkArgs &a, int col0, int qt, ChunkTile &t) {
    t.col0 = col0;
    t.p0 = t.ctx - t.rows;
    t.keys = a.causal ? max(t.p0 + chunk_row_of(a, min(t.col0 + qt, t.cols) - 1) + 1, 0) : t.ctx;
}

__device__ __forceinline__ bool chunk_find_tile(const ChunkArgs &a, int slot, int qt, ChunkTile &t) {
    const int lane = lane_id();
    t.seq = -1;
    for (int s0 = 0; s0 < a.n_seq; s0 += kWave) {
        const int s = min(s0 + lane, a.n_seq - 1);
        const int r0 = a.cu_seqlens[s], r1 = a.cu_seqlens[s + 1], ctx = a.ctx_lens[s];
        const int row0 = chunk_clamp_row(r0, a.total_rows);
        const uint64_t m = __builtin_amdgcn_ballot_w64(s0 + lane < a.n_seq && row0 * a.group / qt + s <= slot);
        if (m != 0) {
            const int at = __builtin_popcountll(m) - 1;
            t.seq = s0 + at;
            t.row0 = __builtin_amdgcn_readlane(row0, at);
            t.rows = max(chunk_clamp_row(__builtin_amdgcn_readlane(r1, at), a.total_rows) - t.row0, 0);
            t.ctx = min(max(__builtin_amdgcn_readlane(ctx, at), 0), a.max_blocks * a.block_size);
        }
        if (m != ~0ull) break;
    }
    if (t.seq < 0) return false;
    t.cols = t.rows * a.group;
    const int n_tiles = (t.cols + qt - 1) / qt;
    const int tile = slot - (t.row0 * a.group / qt + t.seq);
    if (tile < 0 || tile >= n_tiles) return false;
    chunk_tile_at(a, (a.causal ? n_tiles - 1 - tile : tile) * qt, qt, t);   // causal: the tiles with the longest key loops start first
    return true;
}

// Keys per range of a tile that can see `keys` keys, when up to z workgroups share it: a range has `min_keys` keys or
// more, a multiple of bn.
__device__ __forceinline__ int chunk_range_keys(int keys, int z, int bn, int min_keys) {
    const int per = (keys + z - 1) / z;
    return max((per + bn - 1) / bn * bn, min_keys);
}

__device__ __forceinline__ float4_t chunk_mfma16(half8_t a, half8_t b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <int MODE>
__device__ __forceinline__ half8_t chunk_dec8(uint32_t w0, uint32_t w1) {
    u32x4 r;
    uint32_t a, b;
    dec_word<MODE>(w0, a, b);
    r.x = a; r.y = b;
    dec_word<MODE>(w1, a, b);
    r.z = a; r.w = b;
    return __builtin_bit_cast(half8_t, r);
}

// bytes of w whose E5M2 code is infinite or NaN, as 0xFF bytes (E4M3 codes all decode to finite values)
__device__ __forceinline__ uint32_t chunk_nonfinite(uint32_t w) {
    const uint32_t m = ((w & 0x7C7C7C7Cu) + 0x04040404u) & 0x80808080u;
    return (m >> 7) * 0xFFu;
}

__device__ __forceinline__ uint32_t chunk_block_of(const ChunkArgs &a, int pos) {
    return __umulhi(2u * (uint32_t)pos, a.div_mul) >> a.div_shift;
}

// four consecutive dims of one (row, head), starting at dim 4 * w4
template <int D, int MODE>
__device__ __forceinline__ void chunk_store(const ChunkArgs &a, int64_t item, int w4, float4_t x) {
    if (a.out_kind == FEATHER_CHUNK_OUT_F32) {
        *reinterpret_cast<float4_t *>(static_cast<float *>(a.out) + item * D + 4 * w4) = x;
    } else if (a.out_kind == FEATHER_CHUNK_OUT_F16) {
        const half4_t h = {(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
        *reinterpret_cast<half4_t *>(static_cast<_Float16 *>(a.out) + item * D + 4 * w4) = h;
    } else {
        static_cast<uint32_t *>(a.out)[item * (D / 4) + w4] = quant4<MODE>(x[0], x[1], x[2], x[3]);
    }
}

// Rows that belong to no sequence (before cu[0], from cu[n_seq] on): zero, by workgroup `part` of `parts`.
template <int D>
__device__ __forceinline__ void chunk_fill_outside(const ChunkArgs &a, int part, int parts, int threads) {
    const int first = a.n_seq > 0 ? chunk_clamp_row(a.cu_seqlens[0], a.total_rows) : a.total_rows;
    const int last = a.n_seq > 0 ? max(chunk_clamp_row(a.cu_seqlens[a.n_seq], a.total_rows), first) : a.total_rows;
    const int64_t unit = (int64_t)a.n_q_heads * D / 4;                     // packed words of a row
    const int words = a.out_kind == FEATHER_CHUNK_OUT_F32 ? 4 : (a.out_kind == FEATHER_CHUNK_OUT_F16 ? 2 : 1);
    uint32_t *out = static_cast<uint32_t *>(a.out);
    for (int64_t i = (int64_t)part * threads + threadIdx.x; i < (first + (int64_t)(a.total_rows - last)) * unit * words;
         i += (int64_t)parts * threads) {
        const int64_t at = i < first * unit * words ? i : i + (int64_t)(last - first) * unit * words;
        out[at] = 0u;
    }
}

constexpr int kChunkFillGroups = 8;    // workgroups of a grid that only look after rows outside every sequence
// A key range is not cut below this.  LDS kernel: 3 x 97 to 203 rows over 750 to 1501 keys, d = 256: 128 keys 34.5 + 7.6 us
// (kernel, merge), 256 keys 28.6 + 6.2, 512 keys 37.8 + 4.8.  Narrow kernel: two requests of 211 to 300 keys are done in
// one range and one launch, 6.4 us; with ranges of 256 keys 6.3 + 3.6.
constexpr int kChunkMinKeys = 256;
constexpr int kNarrowMinKeys = 512;
constexpr int kNarrowStep = 128;       // keys that the four waves of a narrow workgroup take per turn

// Least keys per range of the narrow kernel: the keys of all its tiles shared out evenly over the workgroups that the
// chip holds at once (less one per tile, for the ranges that a tile ends with), so that a long context is cut into more
// ranges than a short one and the workgroups end together.  Every wave computes it from the lengths; the merge reads it
// from the workspace.
__device__ __forceinline__ int narrow_min_keys(const ChunkArgs &a, int qt) {
    float keys = 0.f;       // an estimate will do
    for (int s = lane_id(); s < a.n_seq; s += kWave) {
        const int rows = max(chunk_clamp_row(a.cu_seqlens[s + 1], a.total_rows) - chunk_clamp_row(a.cu_seqlens[s], a.total_rows), 0);
        const int cols = rows * a.group;
        if (cols <= a.col_split) keys += (float)((cols + qt - 1) / qt) * (float)min(max(a.ctx_lens[s], 0), a.max_blocks * a.block_size);
    }
    const float sum = as_float(__builtin_amdgcn_readfirstlane(as_u32(wave_sum(keys))));
    const int per = __builtin_amdgcn_readfirstlane((int)fminf(sum * a.per_group, 1.0e9f));
    return max((per / kNarrowStep + 1) * kNarrowStep, kNarrowMinKeys);
}

// A column's P = 2^((s - m) c + kShift) refers to a point m that need not be its maximum: O / l does not depend on it, nor
// on kShift, which is the same in every wave and range.  A lane's P are positive, so a sum below kGuard bounds each of them
// by fp16's largest value, 65504; 32 P of 2^kShift sum to 2^13, so a column's scores can grow by a factor of 2^2.9 (all
// equal) to 2^7.9 (one large) before the reference is raised.
constexpr float kShift = 8.f, kGuard = 61440.f;
constexpr float kLazy = 7.f;           // the kernel that compares maxima raises the reference beyond 2^kLazy: P to 2^(kShift + kLazy) = 32768
__device__ __forceinline__ float chunk_reference(float m, float scale_log2e) { return __builtin_fmaf(m, scale_log2e, -kShift); }
// The exponent is one fused operation, s c - (m c - kShift), whose second operand is rounded: by 2^-10 at kFar, by more than 16
// for the largest E5M2 codes, where P of the maximum itself would overflow or vanish.  Columns whose reference is beyond kFar
// subtract the maximum first, (s - m) c + kShift, one operation more: they take the path of a raised reference with every
// tile.  The 16x16 LDS kernel (d = 256, 512), which LDS reads bound, always subtracts first (0 to 1 % of its time).
constexpr float kFar = 16384.f;
template <bool FAR>
__device__ __forceinline__ float chunk_exp(float s, float scale_log2e, float ref) {   // ref: the maximum (FAR), or as chunk_reference gives it
    return __builtin_amdgcn_exp2f(FAR ? __builtin_fmaf(s - ref, scale_log2e, kShift) : __builtin_fmaf(s, scale_log2e, -ref));
}
constexpr int kAnyColumns = 1 << 30;   // more columns than a call can have

// ---- tiles through LDS --------------------------------------------------------------------------------------------
// One workgroup (WAVES waves) owns 16 * QB * WAVES columns, each wave 16 * QB of them for the whole key loop.  Tiles
// of BN keys are fetched packed through the block table into registers two tiles ahead (their block ids three tiles
// ahead: a table entry is never waited for), decoded into the other LDS buffer one tile ahead, and read by all waves.
// PAGE16 (block_size % 16 == 0, the rule of all kernels here): four keys from a multiple of four on share a block, one table
// lookup.  (Multiples of four would do; block sizes like 12 and 20 take the general path.)
template <int D, int MODE, int QB, int BN, int WAVES, bool PAGE16, bool ZS>
__device__ __forceinline__ void chunk_attn_body(const ChunkArgs &a, int bid) {
    constexpr int DW = D / 4;
    constexpr bool BF8 = MODE == FEATHER_E5M2;
    constexpr int KS = BF8 ? (D + 16) / 2 : D + 8;   // K row pitch in LDS, in fp16 units (bf8: D + 16 bytes)
    constexpr int VS = BN, CH = BN / 8;
    constexpr int kThreads = 64 * WAVES, QT = 16 * QB * WAVES;
    constexpr int UNITS = BN * D / 16;
    constexpr int NU = UNITS / kThreads;
    static_assert(UNITS % kThreads == 0 && NU >= 1, "tile / workgroup mismatch");
    constexpr int DB = D / 16, STEPS = D / 32, KB16 = BN / 16, KB32 = BN / 32;
    constexpr int kBufHalfs = BN * KS + D * VS;

    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    _Float16 *const lds = reinterpret_cast<_Float16 *>(smem);
    auto swz = [](int row) { return (row ^ (row >> 2)) & (CH - 1); };

    // Launch order goes round the XCDs (own L2 each): with the KV head fastest an XCD keeps to few heads, and with the tiles
    // slowest the longest tiles of all heads start first on all of them.
    const int kvh = bid % a.n_kv_heads;
    bid /= a.n_kv_heads;
    int zr = 0;
    if constexpr (ZS) {
        zr = bid % a.z_wide;
        bid /= a.z_wide;
    }
    ChunkTile t;
    if (!chunk_find_tile(a, bid, QT, t)) return;
    if (t.cols <= a.col_split) return;                 // a short run of rows: the other kernel's work

    int key_begin = 0, key_end = t.keys;
    if constexpr (ZS) {
        const int per = chunk_range_keys(t.keys, a.z_wide, BN, kChunkMinKeys);
        key_begin = zr * per;
        key_end = min(t.keys, key_begin + per);
        if (key_begin >= key_end) return;              // the merge knows which ranges exist
    }

    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int j = lane & 15, kb = lane >> 4;
    const int qc0 = t.col0 + wave * (16 * QB);         // the wave's first column
    const int32_t *bt = a.block_tables + (int64_t)t.seq * a.max_blocks;
    const int head_rows = kvh * a.block_size, block_rows = a.n_kv_heads * a.block_size;

    // this lane's columns: their row / head, and the last key each sees
    int64_t item[QB];
    int last[QB];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        const int c = min(qc0 + 16 * b + j, t.cols - 1), r = chunk_row_of(a, c);
        item[b] = (int64_t)(t.row0 + r) * a.n_q_heads + kvh * a.group + (c - r * a.group);
        last[b] = a.causal ? t.p0 + r : t.ctx - 1;
    }
    const int wave_first = a.causal ? t.p0 + chunk_row_of(a, min(qc0, t.cols - 1)) : t.ctx - 1;     // smallest and largest last key of the wave
    const int wave_last = a.causal ? t.p0 + chunk_row_of(a, min(qc0 + 16 * QB - 1, t.cols - 1)) : t.ctx - 1;
    const int tile_first = a.causal ? t.p0 + chunk_row_of(a, t.col0) : t.ctx - 1;
    const bool wave_has = qc0 < t.cols;

    half8_t qf[BF8 ? 1 : QB][BF8 ? 1 : STEPS];
    long qf8[BF8 ? QB : 1][BF8 ? STEPS : 1];
#pragma unroll
    for (int b = 0; b < QB; b++)
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(a.q + item[b] * DW + 8 * s + 2 * kb);
            if constexpr (BF8) qf8[b][s] = __builtin_bit_cast(long, w);
            else qf[b][s] = chunk_dec8<MODE>(w.x, w.y);
        }

    float4_t o[QB][DB];
    float m_run[QB], l_run[QB];      // reference point, the lane's share of the sum
#pragma unroll
    for (int b = 0; b < QB; b++) {
        m_run[b] = -INFINITY;
        l_run[b] = 0.f;
#pragma unroll
        for (int d = 0; d < DB; d++) o[b][d] = float4_t{0.f, 0.f, 0.f, 0.f};
    }

    u32x4 kreg[NU];
    uint32_t vreg[NU][4];
    int kid[NU], vid[NU][PAGE16 ? 1 : 4];
    auto fetch_ids = [&](int key0) {
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int u = tid + kThreads * i;
            kid[i] = bt[chunk_block_of(a, min(key0 + u / (D / 16), key_end - 1))];
#pragma unroll
            for (int r = 0; r < (PAGE16 ? 1 : 4); r++)
                vid[i][r] = bt[chunk_block_of(a, min(key0 + 4 * (u / DW) + r, key_end - 1))];
        }
    };
    auto row_of = [&](int id, int pos) {               // cache row in 32 bits (the host checks that every row fits)
        const uint32_t slot = (uint32_t)pos - chunk_block_of(a, pos) * (uint32_t)a.block_size;
        return (int64_t)(uint32_t)(min((uint32_t)id, a.max_blk) * (uint32_t)block_rows + (uint32_t)head_rows + slot);
    };
    auto prefetch = [&](int key0) {                    // the ids of this tile are in kid / vid
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int u = tid + kThreads * i;
            const int kp = key0 + u / (D / 16), c16 = u % (D / 16);
            kreg[i] = u32x4{0, 0, 0, 0};
            if (kp < key_end) kreg[i] = *reinterpret_cast<const u32x4 *>(a.k_cache + row_of(kid[i], kp) * DW + 4 * c16);
            const int ddw = u % DW, vp = key0 + 4 * (u / DW);
            if constexpr (PAGE16) {
                const uint32_t *vr = a.v_cache + row_of(vid[i][0], min(vp, key_end - 1) & ~3) * DW + ddw;
#pragma unroll
                for (int r = 0; r < 4; r++) vreg[i][r] = vp + r < key_end ? vr[r * DW] : 0u;
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++) vreg[i][r] = vp + r < key_end ? a.v_cache[row_of(vid[i][r], vp + r) * DW + ddw] : 0u;
            }
        }
    };
    // decodes the fetched tile into LDS buffer `buf`; returns whether a V code of a tile on the diagonal is infinite or
    // NaN.  Such a code is staged as zero: a column that does not see its key has P = 0 there, and 0 * inf is NaN.
    auto stage = [&](int buf, bool diag) -> int {
        int nf = 0;
        _Float16 *k_lds = lds + buf * kBufHalfs;
        _Float16 *vt_lds = k_lds + BN * KS;
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int u = tid + kThreads * i;
            const int key = u / (D / 16), c16 = u % (D / 16);
            if constexpr (BF8) {
                *reinterpret_cast<u32x4 *>(reinterpret_cast<unsigned char *>(k_lds) + key * (2 * KS) + 16 * c16) = kreg[i];
            } else {
                half8_t *kd = reinterpret_cast<half8_t *>(k_lds + key * KS + 16 * c16);
                kd[0] = chunk_dec8<MODE>(kreg[i].x, kreg[i].y);
                kd[1] = chunk_dec8<MODE>(kreg[i].z, kreg[i].w);
            }
            // V: 4 keys x 4 dims -> V^T[dim][pos]; slot (kb, 4a + r) of a group of 32 keys holds key 16a + 4kb + r
            const int ddw = u % DW, kg = u / DW;
            const int ko = 4 * kg, o32 = ko & 31;
            const int pos = (ko & ~31) + ((o32 & 15) >> 2) * 8 + (o32 >> 4) * 4;
            uint32_t lo2[4], hi2[4];
            if constexpr (BF8) {
                if (diag) {
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t m = chunk_nonfinite(vreg[i][r]);
                        vreg[i][r] &= ~m;
                        nf |= m != 0;
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const uint32_t sel = 0x000c000cu | ((uint32_t)c << 8) | ((uint32_t)(4 + c) << 24);
                    lo2[c] = perm(vreg[i][1], vreg[i][0], sel);
                    hi2[c] = perm(vreg[i][3], vreg[i][2], sel);
                }
            } else {
                uint32_t p01[4], p23[4];
#pragma unroll
                for (int r = 0; r < 4; r++) dec_word<MODE>(vreg[i][r], p01[r], p23[r]);
                lo2[0] = perm(p01[1], p01[0], 0x05040100u); hi2[0] = perm(p01[3], p01[2], 0x05040100u);
                lo2[1] = perm(p01[1], p01[0], 0x07060302u); hi2[1] = perm(p01[3], p01[2], 0x07060302u);
                lo2[2] = perm(p23[1], p23[0], 0x05040100u); hi2[2] = perm(p23[3], p23[2], 0x05040100u);
                lo2[3] = perm(p23[1], p23[0], 0x07060302u); hi2[3] = perm(p23[3], p23[2], 0x07060302u);
            }
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int row = 4 * ddw + c;
                *reinterpret_cast<u32x2 *>(vt_lds + row * VS + (((pos >> 3) ^ swz(row)) << 3) + (pos & 4)) = u32x2{lo2[c], hi2[c]};
            }
        }
        return nf;
    };
    auto on_diag = [&](int key0) { return min(key0 + BN, key_end) - 1 > tile_first; };   // some column does not see some key of the tile

    int nf = 0;
    if (key_begin < key_end) {
        fetch_ids(key_begin);
        prefetch(key_begin);
        fetch_ids(key_begin + BN);
        nf = stage(0, on_diag(key_begin));
        if (key_begin + BN < key_end) {
            prefetch(key_begin + BN);
            fetch_ids(key_begin + 2 * BN);
        }
    }
    if (BF8 && key_begin < key_end && on_diag(key_begin)) nf = __syncthreads_or(nf);
    else __syncthreads();
    int cur = 0;
    for (int key0 = key_begin; key0 < key_end; key0 += BN, cur ^= 1) {
        int nf_next = 0;
        if (key0 + BN < key_end) {
            nf_next = stage(cur ^ 1, on_diag(key0 + BN));
            if (key0 + 2 * BN < key_end) {
                prefetch(key0 + 2 * BN);
                fetch_ids(key0 + 3 * BN);
            }
        }
        const _Float16 *k_lds = lds + cur * kBufHalfs;
        const _Float16 *vt_lds = k_lds + BN * KS;
        const bool masked = key0 + BN - 1 > wave_first;          // wave-uniform: some column does not see some key
        if (wave_has && key0 <= wave_last) {
            half8_t pf[QB][KB32];
            float4_t s[QB][KB16];
#pragma unroll
            for (int c = 0; c < KB16; c++)
#pragma unroll
                for (int st = 0; st < STEPS; st++) {
                    const float4_t zero = {0.f, 0.f, 0.f, 0.f};
                    if constexpr (BF8) {
                        const long kf = *reinterpret_cast<const long *>(reinterpret_cast<const unsigned char *>(k_lds) +
                                                                       (16 * c + j) * (2 * KS) + 32 * st + 8 * kb);
#pragma unroll
                        for (int b = 0; b < QB; b++)
                            s[b][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf8_bf8(kf, qf8[b][st], st == 0 ? zero : s[b][c], 0, 0, 0);
                    } else {
                        const half8_t kf = *reinterpret_cast<const half8_t *>(k_lds + (16 * c + j) * KS + 32 * st + 8 * kb);
#pragma unroll
                        for (int b = 0; b < QB; b++) s[b][c] = chunk_mfma16(kf, qf[b][st], st == 0 ? zero : s[b][c]);
                    }
                }
            mfma_settle<QB * KB16>(&s[0][0]);   // the first readers are asm statements
#pragma unroll
            for (int b = 0; b < QB; b++) {
                if (masked) {
                    int rel = last[b] - key0 - 4 * kb;           // key 16 c + 4 kb + r is hidden if 16 c + r > rel
                    asm volatile("" : "+v"(rel));
#pragma unroll
                    for (int c = 0; c < KB16; c++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            if (16 * c + r > rel) s[b][c][r] = -INFINITY;
                }
                float mx = max3_raw(s[b][0][0], s[b][0][1], s[b][0][2]);
                mx = max_raw(mx, s[b][0][3]);
#pragma unroll
                for (int c = 1; c < KB16; c++) {
                    mx = max3_raw(mx, s[b][c][0], s[b][c][1]);
                    mx = max3_raw(mx, s[b][c][2], s[b][c][3]);
                }
                mx = max_xor32(max_xor16(mx));
                // m_run is the point that P refers to, kShift below the maximum (at it where the scores are so large that the
                // difference would be rounded up).  It is raised only when a column exceeds it by 2^(kShift + kLazy).  A
                // column that has seen no key yet keeps -inf and refers to zero: its scores are -inf, its P zero.
                const float m_old = m_run[b];
                const bool raise = __builtin_amdgcn_ballot_w64(mx - m_old > a.raise_raw) != 0;
                const float low = mx - a.shift_raw, m_new = raise ? max_raw(m_old, mx - low > 1.1f * a.shift_raw ? mx : low) : m_old;
                const float ref = m_new == -INFINITY ? 0.f : m_new;
                if (raise) {
                    const float alpha = m_old == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_old - m_new) * a.scale_log2e);
                    m_run[b] = m_new;
                    l_run[b] *= alpha;
#pragma unroll
                    for (int d = 0; d < DB; d++) o[b][d] *= alpha;
                }
#pragma unroll
                for (int g = 0; g < KB32; g++) {
                    uint32_t pw[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float4_t &x = s[b][2 * g + (i >> 1)];
                        const float e0 = __builtin_amdgcn_exp2f((x[2 * (i & 1)] - ref) * a.scale_log2e);   // (subtracted first: see kFar)
                        const float e1 = __builtin_amdgcn_exp2f((x[2 * (i & 1) + 1] - ref) * a.scale_log2e);
                        pw[i] = as_u32(__builtin_convertvector(float2p_t{e0, e1}, half2_t));
                        l_run[b] = dot2(pw[i], 0x3c003c00u, l_run[b]);   // the sum takes the rounded values that multiply V
                    }
                    pf[b][g] = __builtin_bit_cast(half8_t, u32x4{pw[0], pw[1], pw[2], pw[3]});
                }
            }
#pragma unroll
            for (int g = 0; g < KB32; g++)
#pragma unroll
                for (int d = 0; d < DB; d++) {
                    const half8_t vf = *reinterpret_cast<const half8_t *>(vt_lds + (16 * d + j) * VS + (((4 * g + kb) ^ swz(16 * d + j)) << 3));
#pragma unroll
                    for (int b = 0; b < QB; b++) o[b][d] = chunk_mfma16(vf, pf[b][g], o[b][d]);
                }
            if (BF8 && nf) {   // rare: what the staged zeros stand for, added for the columns that see the key
                for (int key = key0; key < min(key0 + BN, key_end); key++) {
                    const uint32_t *vr = a.v_cache + row_of(bt[chunk_block_of(a, key)], key) * DW + kb;
#pragma unroll
                    for (int d = 0; d < DB; d++) {
                        const uint32_t w = vr[4 * d];
                        if (chunk_nonfinite(w) != 0) {
                            const uint32_t m = chunk_nonfinite(w);
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const float x = (float)__builtin_bit_cast(_Float16, (uint16_t)((w >> (8 * r)) << 8));
                                if ((m >> (8 * r)) & 1u)
#pragma unroll
                                    for (int b = 0; b < QB; b++)
                                        if (key <= last[b]) o[b][d][r] += x;
                            }
                        }
                    }
                }
            }
        }
        // only a tile on the diagonal can have something to report (the vote costs more than the barrier)
        if (BF8 && key0 + BN < key_end && on_diag(key0 + BN)) {
            nf = __syncthreads_or(nf_next);
        } else {
            nf = 0;
            __syncthreads();
        }
    }

    if (!wave_has) return;
#pragma unroll
    for (int b = 0; b < QB; b++) {
        float l = l_run[b];
        l += __shfl_xor(l, 16, kWave);
        l += __shfl_xor(l, 32, kWave);
        if (qc0 + 16 * b + j >= t.cols) continue;
        if constexpr (ZS) {
            const int64_t items = (int64_t)a.total_rows * a.n_q_heads, at = zr * items + item[b];
#pragma unroll
            for (int d = 0; d < DB; d++) *reinterpret_cast<float4_t *>(a.part + at * D + 16 * d + 4 * kb) = o[b][d];
            if (kb == 0) *reinterpret_cast<float2p_t *>(a.part + a.z_wide * items * D + at * 2) = float2p_t{m_run[b], l};
        } else {
            const float inv = l == 0.f ? 0.f : 1.0f / l;          // no visible key: a zero result
#pragma unroll
            for (int d = 0; d < DB; d++) chunk_store<D, MODE>(a, item[b], 4 * d + kb, l == 0.f ? float4_t{0.f, 0.f, 0.f, 0.f} : o[b][d] * inv);
        }
    }
}

// ---- tiles through LDS on the 32x32 matrix instructions -----------------------------------------------------------------
// The split and the numerics of chunk_attn_body, and the instruction mix of the prefill kernel's d = 64 form: vector
// issue bounds these head dims, and an instruction of 32x32 holds it half as long per product as two of 16x16 --
//     S^T[32 keys, 32 cols] = v_mfma_f32_32x32x64_f8f6f4 (E5M2 bytes as they are: the whole head dim) or four of
//                             v_mfma_f32_32x32x16_f16 (E4M3, decoded);   O^T[32 dims, 32 cols] += v_mfma_f32_32x32x16_f16
// A wave owns 32 * CB columns.  Lane l: n = l % 32 the column, h = l / 32; accumulator register r is row
// 8 (r / 4) + 4 h + r % 4.  Registers 8 s .. 8 s + 7 of the scores are the k-slots of the second product's step s if V^T
// holds the keys of every group of 16 in the order 0 1 2 3 8 9 10 11 | 4 5 6 7 12 13 14 15.
// PAGE16 (block_size % 16 == 0): the 16 keys that a wave stages share a block, whose address is then scalar.
// Against chunk_attn_body: d = 64, E5M2, the chunk of 2048 rows above 320 -> 155 us; d = 128, 512 rows over 4000 keys
// 42 -> 33 us; d = 256 (4 waves of 32 columns, one wave per SIMD) 28 -> 48 us, so that one stays.
typedef int int8p_t __attribute__((ext_vector_type(8)));

template <int D, int MODE, int CB, int WAVES, bool PAGE16, bool ZS>
__device__ __forceinline__ void chunk_attn32_body(const ChunkArgs &a, int bid) {
    constexpr bool BF8 = MODE == FEATHER_E5M2;
    constexpr int DW = D / 4, BN = 64, DB = D / 32, STEPS = BF8 ? D / 64 : D / 16;   // 32-dim blocks; matrix steps of a score block
    constexpr int KP = (BF8 ? D : 2 * D) + 16;   // K row pitch in LDS, bytes
    constexpr int VS = BN;                       // fp16 per V^T row
    constexpr int kThreads = 64 * WAVES, QT = 32 * CB * WAVES;
    constexpr int kBufBytes = BN * KP + D * VS * 2;
    constexpr int UNITS = BN * D / 16, NU = UNITS / kThreads;
    static_assert(UNITS % kThreads == 0 && NU >= 1, "tile / workgroup mismatch");

    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    auto swz = [](int row) { return ((row >> 1) & 7) ^ ((row >> 4) & 1); };   // 16-byte chunk c of V^T row r lives at chunk c ^ swz(r)

    // Launch order goes round the XCDs (own L2 each): with the KV head fastest an XCD keeps to few heads, and with the tiles
    // slowest the longest tiles of all heads start first on all of them.
    const int kvh = bid % a.n_kv_heads;
    bid /= a.n_kv_heads;
    int zr = 0;
    if constexpr (ZS) {
        zr = bid % a.z_wide;
        bid /= a.z_wide;
    }
    ChunkTile t;
    if (!chunk_find_tile(a, bid, QT, t)) return;
    if (t.cols <= a.col_split) return;                 // a short run of rows: the other kernel's work
    int key_begin = 0, key_end = t.keys;
    if constexpr (ZS) {
        const int per = chunk_range_keys(t.keys, a.z_wide, BN, kChunkMinKeys);
        key_begin = zr * per;
        key_end = min(t.keys, key_begin + per);
        if (key_begin >= key_end) return;              // the merge knows which ranges exist
    }

    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
    const int n = lane & 31, h = lane >> 5;
    const int qc0 = t.col0 + wave * (32 * CB);
    const int32_t *bt = a.block_tables + (int64_t)t.seq * a.max_blocks;
    const uint32_t block_bytes = (uint32_t)(a.n_kv_heads * a.block_size) * D;
    const int64_t head_bytes = (int64_t)kvh * a.block_size * D;
    auto slot_of = [&](int pos) { return (uint32_t)pos - chunk_block_of(a, pos) * (uint32_t)a.block_size; };
    auto row_at = [&](const uint32_t *cache, int id, int pos) {
        return reinterpret_cast<const char *>(cache) + ((uint64_t)min((uint32_t)id, a.max_blk) * block_bytes + (uint64_t)head_bytes + slot_of(pos) * D);
    };

    int64_t item[CB];
    int last[CB];
#pragma unroll
    for (int b = 0; b < CB; b++) {
        const int c = min(qc0 + 32 * b + n, t.cols - 1), r = chunk_row_of(a, c);
        item[b] = (int64_t)(t.row0 + r) * a.n_q_heads + kvh * a.group + (c - r * a.group);
        last[b] = a.causal ? t.p0 + r : t.ctx - 1;
    }
    const int wave_first = a.causal ? t.p0 + chunk_row_of(a, min(qc0, t.cols - 1)) : t.ctx - 1;
    const int wave_last = a.causal ? t.p0 + chunk_row_of(a, min(qc0 + 32 * CB - 1, t.cols - 1)) : t.ctx - 1;
    const int tile_first = a.causal ? t.p0 + chunk_row_of(a, t.col0) : t.ctx - 1;
    const bool wave_has = qc0 < t.cols;

    int8p_t qf[BF8 ? CB : 1][BF8 ? STEPS : 1];
    half8_t qh16[BF8 ? 1 : CB][BF8 ? 1 : STEPS];
#pragma unroll
    for (int b = 0; b < CB; b++) {
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            if constexpr (BF8) {
                const u32x2 *src = reinterpret_cast<const u32x2 *>(a.q + item[b] * DW + 16 * st + 8 * h);   // q need not be aligned to 16 bytes
                const u32x2 w0 = src[0], w1 = src[1], w2 = src[2], w3 = src[3];
                qf[b][st] = int8p_t{(int)w0.x, (int)w0.y, (int)w1.x, (int)w1.y, (int)w2.x, (int)w2.y, (int)w3.x, (int)w3.y};
            } else {
                const u32x2 w = *reinterpret_cast<const u32x2 *>(a.q + item[b] * DW + 4 * st + 2 * h);
                qh16[b][st] = chunk_dec8<MODE>(w.x, w.y);
            }
        }
    }

    float16_t o[CB][DB];                         // [32-dim block]
    float m_run[CB], mc_run[CB], l_run[CB];      // reference point (raw, and as chunk_reference gives it), the lane's share of the sum
#pragma unroll
    for (int b = 0; b < CB; b++) {
        m_run[b] = mc_run[b] = -INFINITY;
        l_run[b] = 0.f;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[b][d][r] = 0.f;
    }

    // ---- staging: a thread carries NU units of K (16 bytes of one key) and of V (4 keys x 4 dims); unit u of either is in
    // the keys u / (D / 16) .. of the tile, so the 64 units of a wave lie in 16 neighbouring keys, the same for K and V
    const int key_wave = wave * (1024 / D);      // the wave's first key of its first units
    constexpr int kKeysPerTurn = kThreads * 16 / D;
    const __attribute__((address_space(4))) int32_t *bt_const = (const __attribute__((address_space(4))) int32_t *)bt;   // read only while the kernel runs: scalar loads
    int id_k[NU], id_v[PAGE16 ? 1 : NU][PAGE16 ? 1 : 4];   // PAGE16: id_k only, wave-uniform
    auto first16 = [&](int key0, int i) { return min((key0 + key_wave + kKeysPerTurn * i) & ~15, (key_end - 1) & ~15); };
    auto fetch_ids = [&](int key0) {
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int u = tid + kThreads * i;
            if constexpr (PAGE16) {
                id_k[i] = bt_const[chunk_block_of(a, first16(key0, i))];
            } else {
                id_k[i] = bt[chunk_block_of(a, min(key0 + u / (D / 16), key_end - 1))];
#pragma unroll
                for (int r = 0; r < 4; r++) id_v[i][r] = bt[chunk_block_of(a, min(key0 + 4 * (u / DW) + r, key_end - 1))];
            }
        }
    };
    u32x4 kreg[NU];
    uint32_t vreg[NU][4];
    auto prefetch = [&](int key0) {              // keys past the end: another key's row (masked; its V is zeroed by `stage`)
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int u = tid + kThreads * i;
            if constexpr (PAGE16) {
                const int pos = first16(key0, i);
                kreg[i] = *reinterpret_cast<const u32x4 *>(row_at(a.k_cache, id_k[i], pos) + (uint32_t)((u / (D / 16) % 16) * D + 16 * (u % (D / 16))));
                const char *vr = row_at(a.v_cache, id_k[i], pos) + (uint32_t)((u / DW % 4) * 4 * D + 4 * (u % DW));
#pragma unroll
                for (int r = 0; r < 4; r++) vreg[i][r] = *reinterpret_cast<const uint32_t *>(vr + r * D);
            } else {
                kreg[i] = *reinterpret_cast<const u32x4 *>(row_at(a.k_cache, id_k[i], min(key0 + u / (D / 16), key_end - 1)) + 16 * (u % (D / 16)));
#pragma unroll
                for (int r = 0; r < 4; r++)
                    vreg[i][r] = *reinterpret_cast<const uint32_t *>(row_at(a.v_cache, id_v[i][r], min(key0 + 4 * (u / DW) + r, key_end - 1)) + 4 * (u % DW));
            }
        }
    };
    auto on_diag = [&](int key0) { return min(key0 + BN, key_end) - 1 > tile_first; };   // some column does not see some key of the tile
    // decodes the fetched tile into buffer `buf`; E5M2: codes of inf and NaN in V are staged as zero where a column does not
    // see some key of the tile (P = 0 there, and 0 * inf is NaN), and reported
    auto stage = [&](int buf, int key0) -> int {
        int nf = 0;
        unsigned char *k_lds = smem + buf * kBufBytes;
        _Float16 *vt_lds = reinterpret_cast<_Float16 *>(k_lds + BN * KP);
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int u = tid + kThreads * i;
            const int key = u / (D / 16), c16 = u % (D / 16);
            if constexpr (BF8) {
                *reinterpret_cast<u32x4 *>(k_lds + key * KP + 16 * c16) = kreg[i];
            } else {
                half8_t *kd = reinterpret_cast<half8_t *>(k_lds + key * KP + 32 * c16);
                kd[0] = chunk_dec8<MODE>(kreg[i].x, kreg[i].y);
                kd[1] = chunk_dec8<MODE>(kreg[i].z, kreg[i].w);
            }
            const int ddw = u % DW, kg = u / DW;
            const int q4 = kg & 3, pos = 16 * (kg >> 2) + 8 * (q4 & 1) + 4 * (q4 >> 1);
            uint32_t (&w)[4] = vreg[i];
            if (key0 + BN > key_end)
#pragma unroll
                for (int r = 0; r < 4; r++) w[r] = key0 + 4 * kg + r < key_end ? w[r] : 0u;
            uint32_t lo2[4], hi2[4];         // halfs (key 0, key 1) and (key 2, key 3) of dim 4 ddw + c
            if constexpr (BF8) {
                if (on_diag(key0)) {
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t m = chunk_nonfinite(w[r]);
                        w[r] &= ~m;
                        nf |= m != 0;
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const uint32_t sel = 0x000c000cu | ((uint32_t)c << 8) | ((uint32_t)(4 + c) << 24);
                    lo2[c] = perm(w[1], w[0], sel);
                    hi2[c] = perm(w[3], w[2], sel);
                }
            } else {
                uint32_t p01[4], p23[4];
#pragma unroll
                for (int r = 0; r < 4; r++) dec_word<MODE>(w[r], p01[r], p23[r]);
                lo2[0] = perm(p01[1], p01[0], 0x05040100u); hi2[0] = perm(p01[3], p01[2], 0x05040100u);
                lo2[1] = perm(p01[1], p01[0], 0x07060302u); hi2[1] = perm(p01[3], p01[2], 0x07060302u);
                lo2[2] = perm(p23[1], p23[0], 0x05040100u); hi2[2] = perm(p23[3], p23[2], 0x05040100u);
                lo2[3] = perm(p23[1], p23[0], 0x07060302u); hi2[3] = perm(p23[3], p23[2], 0x07060302u);
            }
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int row = 4 * ddw + c;
                *reinterpret_cast<u32x2 *>(vt_lds + row * VS + (((pos >> 3) ^ swz(row)) << 3) + (pos & 4)) = u32x2{lo2[c], hi2[c]};
            }
        }
        return nf;
    };

    int nf = 0;
    if (key_begin < key_end) {
        fetch_ids(key_begin);
        prefetch(key_begin);
        fetch_ids(key_begin + BN);
        nf = stage(0, key_begin);
        if (key_begin + BN < key_end) {
            prefetch(key_begin + BN);
            fetch_ids(key_begin + 2 * BN);
        }
    }
    if (BF8 && key_begin < key_end && on_diag(key_begin)) nf = __syncthreads_or(nf);
    else __syncthreads();
    // one tile; the buffer index is a compile-time constant, so LDS addresses are loop-invariant registers plus immediates
    auto tile_body = [&](const int key0, auto cur_c) {
        constexpr int cur = decltype(cur_c)::value;
        const unsigned char *k_lds = smem + cur * kBufBytes;
        const _Float16 *vt_lds = reinterpret_cast<const _Float16 *>(k_lds + BN * KP);
        int nf_next = 0;
        if (key0 + BN < key_end) {
            nf_next = stage(cur ^ 1, key0 + BN);
            if (key0 + 2 * BN < key_end) {
                prefetch(key0 + 2 * BN);
                fetch_ids(key0 + 3 * BN);
            }
        }
        const bool masked = key0 + BN - 1 > wave_first;           // wave-uniform: some column does not see some key
        if (wave_has && key0 <= wave_last) {
            auto v_frag = [&](int g, int d) {   // 16-key step, 32-dim block
                const int row = 32 * d + n;
                return *reinterpret_cast<const half8_t *>(vt_lds + row * VS + (((2 * g + h) ^ swz(row)) << 3));
            };
            half8_t vf[4][D == 64 ? 2 : 1];     // d = 64: all of them, requested ahead of the scores
            if constexpr (D == 64)
#pragma unroll
                for (int g = 0; g < 4; g++)
#pragma unroll
                    for (int d = 0; d < 2; d++) vf[g][d] = v_frag(g, d);
            float16_t sc[CB][2];
            const float16_t zero16 = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
                for (int st = 0; st < STEPS; st++) {
                    if constexpr (BF8) {
                        const u32x4 *src = reinterpret_cast<const u32x4 *>(k_lds + (32 * c + n) * KP + 64 * st + 32 * h);
                        const u32x4 w0 = src[0], w1 = src[1];
                        const int8p_t kf = {(int)w0.x, (int)w0.y, (int)w0.z, (int)w0.w, (int)w1.x, (int)w1.y, (int)w1.z, (int)w1.w};
#pragma unroll
                        for (int b = 0; b < CB; b++)   // both operands in the BF8 (E5M2) format, no block scales
                            sc[b][c] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(kf, qf[b][st], st == 0 ? zero16 : sc[b][c], 1, 1, 0, 0, 0, 0);
                    } else {
                        const half8_t k16 = *reinterpret_cast<const half8_t *>(k_lds + (32 * c + n) * KP + 32 * st + 16 * h);
#pragma unroll
                        for (int b = 0; b < CB; b++)
                            sc[b][c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k16, qh16[b][st], st == 0 ? zero16 : sc[b][c], 0, 0, 0);
                    }
                }
            half8_t pb[CB][4];
#pragma unroll
            for (int b = 0; b < CB; b++) {
                if (masked) {
                    int rel = last[b] - key0 - 4 * h;             // key 32 c + 8 (r / 4) + 4 h + r % 4 is hidden if 32 c + 8 (r / 4) + r % 4 > rel
                    asm volatile("" : "+v"(rel));                 // keeps the 32 compares inside this rarely taken branch
#pragma unroll
                    for (int c = 0; c < 2; c++)
#pragma unroll
                        for (int r = 0; r < 16; r++)
                            if (32 * c + 8 * (r >> 2) + (r & 3) > rel) sc[b][c][r] = -INFINITY;
                }
                // P against the column's current reference point; the lane's share of the sum tells whether that was safe
                // (see kGuard); if not, the reference is raised to the true maximum and P computed again
                auto exp_block = [&](auto far_c, const float ref) {
                    constexpr bool FAR = decltype(far_c)::value;
                    float sum = 0.f;
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        uint32_t pw[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float e0 = chunk_exp<FAR>(sc[b][g >> 1][8 * (g & 1) + 2 * i], a.scale_log2e, ref);
                            const float e1 = chunk_exp<FAR>(sc[b][g >> 1][8 * (g & 1) + 2 * i + 1], a.scale_log2e, ref);
                            pw[i] = as_u32(__builtin_convertvector(float2p_t{e0, e1}, half2_t));
                            sum = dot2(pw[i], 0x3c003c00u, sum);  // the sum takes the rounded values that multiply V
                        }
                        pb[b][g] = __builtin_bit_cast(half8_t, u32x4{pw[0], pw[1], pw[2], pw[3]});
                    }
                    return sum;
                };
                float sum = exp_block(std::false_type{}, mc_run[b]);
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(sum < kGuard)) != 0, 0)) {
                    float mx = max3_raw(sc[b][0][0], sc[b][0][1], sc[b][0][2]);
                    mx = max_raw(mx, sc[b][0][3]);
#pragma unroll
                    for (int i = 2; i < 16; i++) mx = max3_raw(mx, sc[b][i >> 3][(2 * i) & 15], sc[b][i >> 3][(2 * i + 1) & 15]);
                    mx = max_xor32(mx);                           // the two lanes of a column
                    const float m_old = m_run[b], m_new = max_raw(m_old, mx);
                    // a column that has seen no key keeps the reference -inf: its scores are -inf here, its P zero
                    const float alpha = m_old == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_old - m_new) * a.scale_log2e);
                    const float mc = chunk_reference(m_new, a.scale_log2e);
                    const bool far = m_new != -INFINITY && __builtin_fabsf(mc) > kFar;
                    m_run[b] = m_new;
                    mc_run[b] = far ? -INFINITY : mc;             // (-inf: such a column comes here with every tile)
                    l_run[b] *= alpha;
#pragma unroll
                    for (int d = 0; d < DB; d++) o[b][d] *= alpha;
                    if (__builtin_amdgcn_ballot_w64(far) != 0) sum = exp_block(std::true_type{}, m_new == -INFINITY ? 0.f : m_new);
                    else sum = exp_block(std::false_type{}, m_new == -INFINITY ? 0.f : mc);
                }
                l_run[b] += sum;
                if constexpr (D == 64)
#pragma unroll
                    for (int g = 0; g < 4; g++)
#pragma unroll
                        for (int d = 0; d < 2; d++) o[b][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[g][d], pb[b][g], o[b][d], 0, 0, 0);
            }
            if constexpr (D > 64)
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int g = 0; g < 4; g++) {
                        const half8_t v1 = v_frag(g, d);
#pragma unroll
                        for (int b = 0; b < CB; b++) o[b][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, pb[b][g], o[b][d], 0, 0, 0);
                    }
            if (BF8 && nf) {   // rare: what the staged zeros stand for, added for the columns that see the key
                for (int key = key0; key < min(key0 + BN, key_end); key++) {
                    const uint32_t *vr = reinterpret_cast<const uint32_t *>(row_at(a.v_cache, bt[chunk_block_of(a, key)], key)) + h;
#pragma unroll
                    for (int d = 0; d < DB; d++)
#pragma unroll
                        for (int g = 0; g < 4; g++) {             // dims 32 d + 8 g + 4 h + {0..3}
                            const uint32_t w = vr[8 * d + 2 * g], m = chunk_nonfinite(w);
                            if (m != 0)
#pragma unroll
                                for (int r = 0; r < 4; r++)
                                    if ((m >> (8 * r)) & 1u) {
                                        const float x = (float)__builtin_bit_cast(_Float16, (uint16_t)((w >> (8 * r)) << 8));
#pragma unroll
                                        for (int b = 0; b < CB; b++)
                                            if (key <= last[b]) o[b][d][4 * g + r] += x;
                                    }
                        }
                }
            }
        }
        // only a tile on the diagonal can have something to report (the vote costs more than the barrier)
        if (BF8 && key0 + BN < key_end && on_diag(key0 + BN)) {
            nf = __syncthreads_or(nf_next);
        } else {
            nf = 0;
            __syncthreads();
        }
    };
    for (int key0 = key_begin; key0 < key_end; key0 += 2 * BN) {
        tile_body(key0, std::integral_constant<int, 0>{});
        if (key0 + BN < key_end) tile_body(key0 + BN, std::integral_constant<int, 1>{});
    }

    if (!wave_has) return;
#pragma unroll
    for (int b = 0; b < CB; b++) {
        const float l = l_run[b] + as_float((uint32_t)__builtin_amdgcn_ds_bpermute(4 * (lane ^ 32), (int)as_u32(l_run[b])));
        if (qc0 + 32 * b + n >= t.cols) continue;
        const int64_t items = (int64_t)a.total_rows * a.n_q_heads, at = zr * items + item[b];
        const float inv = l == 0.f ? 0.f : 1.0f / l;              // no visible key: a zero result
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const float4_t x = {o[b][d][4 * g], o[b][d][4 * g + 1], o[b][d][4 * g + 2], o[b][d][4 * g + 3]};
                if constexpr (ZS) *reinterpret_cast<float4_t *>(a.part + at * D + 32 * d + 8 * g + 4 * h) = x;
                else chunk_store<D, MODE>(a, item[b], 8 * d + 2 * g + h, l == 0.f ? float4_t{0.f, 0.f, 0.f, 0.f} : x * inv);
            }
        if constexpr (ZS)
            if (h == 0) *reinterpret_cast<float2p_t *>(a.part + a.z_wide * items * D + at * 2) = float2p_t{m_run[b], l};
    }
}

// ---- few columns: keys straight from the cache ----------------------------------------------------------------------
// A drafted token or a handful of them: few tiles of 16 * NB columns per (sequence, KV head), so the cache is read once or a
// few times and its bytes bound the kernel.  One workgroup of four waves per (tile, KV head, key range); the waves take the range's
// steps of 32 keys in turn and share nothing until the end:
//     S^T[key, col]   = K Q^T       a lane holds 16 codes of one key: the A operand of two products
//     O_c^T[i, col]  += V_c^T P^T   dim = 4 i + c: the lane holds the same word of eight keys and byte c of them is the
//                                   A operand of the c-th product, so V is transposed by the byte select of its decode
// RING > 0 (block_size a multiple of 16, so 16 keys from a multiple of 16 on are in one block): the packed rows go from
// memory to LDS without passing through registers, RING steps of a wave in flight or in use, into a ring of the wave's
// own (no barrier, only the wave's count of outstanding loads).  A load moves 1 KiB with a wave-uniform base -- the block
// id is a scalar load, the address scalar arithmetic -- and the lane's constant offset.  Registers then hold one step
// only.
// RING = 0 (any block size): rows go to registers, NF steps in flight, an address for every key.
// Each wave keeps its own reference point and sums; they are joined through LDS, and the ranges by the merge kernel.
// Measured: 16 rows of 32 heads on 8 at context 65537, d = 128, E4M3 48 + 5 us (E5M2 38 + 5): two tiles of 32 columns, each of
// which requests and decodes the 134 MB of the cache for itself, 2.8 TB/s of different bytes (one tile of 64 columns 45 us, but
// see narrow_blocks); 32 requests with 3 to 8 rows, contexts to 4096, 32 heads on 4, d = 64, E4M3 24 + 5 us for 39 MB: a wave
// has five steps there, and the round trips in front of them (lengths, block ids, rows), the exponentials of 64 columns and
// the join bound it.  Blocks that are no multiples of 16, through registers: blocks of 20 at context 65537 57 + 5 us, the 32
// requests with blocks of 8 or 20 25 + 4 us.
template <int D>
struct NarrowStep {
    u32x4 kw[2][D / 64];
    uint32_t vw[D / 64][2][4];
};

typedef __attribute__((address_space(3))) unsigned char lds_byte;
typedef __attribute__((address_space(1))) unsigned char global_byte;

// K and V of a step from the wave's ring slot.  The reads are asm statements with their wait inside: the compiler does
// not see that they read what the direct loads wrote (it would wait for all of those, not for the step's); the caller
// waits for the step's loads.  A row of D bytes has its 16-byte chunks XORed with row bits, so that the rows a read
// touches fall on different banks.
template <int D>
__device__ __forceinline__ int ring_swizzle(int row) { return D == 64 ? (row >> 1) & 3 : row & 7; }

#define RING_V_OUT(c)                                                                                                   \
    "=&v"(S.vw[c][0][0]), "=&v"(S.vw[c][0][1]), "=&v"(S.vw[c][0][2]), "=&v"(S.vw[c][0][3]), "=&v"(S.vw[c][1][0]),      \
        "=&v"(S.vw[c][1][1]), "=&v"(S.vw[c][1][2]), "=&v"(S.vw[c][1][3])

template <int D>
__device__ __forceinline__ void ring_read(uint32_t slot, uint32_t koff, const uint32_t (&voff)[4], NarrowStep<D> &S) {
    // chunk 4 c + kb of a row: the XOR leaves bits above the swizzle alone, so c moves the address by an XOR of 64 c
#pragma unroll
    for (int c = 0; c < D / 64; c++) {
        const uint32_t x = 64u * c, k0 = slot + (koff ^ x), v0 = slot + (voff[0] ^ x), v1 = slot + (voff[1] ^ x),
                       v2 = slot + (voff[2] ^ x), v3 = slot + (voff[3] ^ x);
        asm volatile("ds_read_b128 %0, %10\n\tds_read_b128 %1, %10 offset:%15\n\t"
                     "ds_read_b32 %2, %11 offset:%16\n\tds_read_b32 %3, %12 offset:%16\n\t"
                     "ds_read_b32 %4, %13 offset:%16\n\tds_read_b32 %5, %14 offset:%16\n\t"
                     "ds_read_b32 %6, %11 offset:%17\n\tds_read_b32 %7, %12 offset:%17\n\t"
                     "ds_read_b32 %8, %13 offset:%17\n\tds_read_b32 %9, %14 offset:%17\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(S.kw[0][c]), "=&v"(S.kw[1][c]), RING_V_OUT(c)
                     : "v"(k0), "v"(v0), "v"(v1), "v"(v2), "v"(v3), "n"(16 * D), "n"(32 * D), "n"(48 * D) : "memory");
    }
}
#undef RING_V_OUT

__device__ __forceinline__ int64_t narrow_items(const ChunkArgs &a) {
    return (a.narrow_rows ? (int64_t)a.n_seq * a.narrow_rows : a.total_rows) * a.n_q_heads;
}
__device__ __forceinline__ int64_t narrow_item(const ChunkArgs &a, int64_t item, int seq, int row0) {
    return a.narrow_rows ? item + ((int64_t)seq * a.narrow_rows - row0) * a.n_q_heads : item;
}

template <int D, int MODE, int NB, int RING>
__device__ __forceinline__ void chunk_narrow_body(const ChunkArgs &a, int pair, int tile, int zr) {
    constexpr int DW = D / 4, RB = D / 64, STEPS = D / 32, QT = 16 * NB, W = 4, STEP = 32;
    constexpr bool BF8 = MODE == FEATHER_E5M2;
    constexpr int NF = RING > 0 ? 1 : (D == 64 ? (NB == 4 ? 2 : 4) : (D == 128 ? 2 : 1));
    static_assert(STEP * W == kNarrowStep, "keys per turn");
    __shared__ float ml_lds[NB][W][2][16];
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    float4_t *const x_lds = reinterpret_cast<float4_t *>(smem);     // [NB][W][RB * 4][64]

    // In launch order, which goes round the XCDs, all first ranges come before all second ones and so on: ranges that do
    // not exist come last.  A workgroup has one tile of its sequence -- unless the caller's bound of the rows was wrong, then
    // it takes others after it.
    const int seq_i = (int)(__umulhi(2u * (uint32_t)pair, a.kv_mul) >> a.kv_shift), kvh = pair - seq_i * a.n_kv_heads;
    ChunkTile t;
    t.seq = seq_i;
    t.row0 = chunk_clamp_row(a.cu_seqlens[seq_i], a.total_rows);
    t.rows = max(chunk_clamp_row(a.cu_seqlens[seq_i + 1], a.total_rows) - t.row0, 0);
    t.cols = t.rows * a.group;
    if (tile > 0 && tile * QT >= t.cols) return;
    t.ctx = min(max(a.ctx_lens[seq_i], 0), a.max_blocks * a.block_size);
    int least = kNarrowMinKeys;
    if (a.z_narrow > 1) {
        least = narrow_min_keys(a, QT);
        if (pair + tile + zr == 0 && threadIdx.x == 0) *reinterpret_cast<int *>(a.part_narrow + narrow_items(a) * a.z_narrow * (D + 2)) = least;
    }
    if (t.cols > a.col_split) return;                               // a long run of rows: the other kernel's work
#pragma nounroll
    for (int col0 = tile * QT; col0 < t.cols; col0 += a.narrow_tiles * QT) {
    chunk_tile_at(a, col0, QT, t);
    const int per = chunk_range_keys(t.keys, a.z_narrow, kNarrowStep, least);
    const int key_begin = zr * per, key_end = min(t.keys, key_begin + per);
    if (key_begin >= key_end && (zr > 0 || a.z_narrow > 1)) continue;   // the merge knows which ranges exist

    const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), j = lane & 15, kb = lane >> 4;
    const int32_t *bt = a.block_tables + (int64_t)t.seq * a.max_blocks;
    const uint32_t block_bytes = (uint32_t)(a.n_kv_heads * a.block_size) * D;      // below 2^31: checked by the host
    const int64_t head_bytes = (int64_t)kvh * a.block_size * D;
    auto slot_of = [&](int pos) { return (uint32_t)pos - chunk_block_of(a, pos) * (uint32_t)a.block_size; };
    auto row_at = [&](const uint32_t *cache, int id, int pos, int byte) {
        return reinterpret_cast<const char *>(cache) + head_bytes + ((uint64_t)min((uint32_t)id, a.max_blk) * block_bytes + (slot_of(pos) * D + byte));
    };

    using Step = NarrowStep<D>;
    struct Ids {
        int k[2], v[2][4];
    };
    Step steps[NF];
    Ids ids[NF];
    const int last_key = key_end - 1;                               // positions past the range repeat its last key (or its neighbours) and are masked
    auto fetch_ids = [&](Ids &I, int t0) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            I.k[h] = bt[chunk_block_of(a, min(t0 + 16 * h + j, last_key))];
#pragma unroll
            for (int r = 0; r < 4; r++) I.v[h][r] = bt[chunk_block_of(a, min(t0 + 16 * h + 4 * kb + r, last_key))];
        }
    };
    auto load_step = [&](Step &S, const Ids &I, int t0) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const char *kr = row_at(a.k_cache, I.k[h], min(t0 + 16 * h + j, last_key), 16 * kb);
#pragma unroll
            for (int c = 0; c < RB; c++) S.kw[h][c] = *reinterpret_cast<const u32x4 *>(kr + 64 * c);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const char *vr = row_at(a.v_cache, I.v[h][r], min(t0 + 16 * h + 4 * kb + r, last_key), 4 * j);
#pragma unroll
                for (int c = 0; c < RB; c++) S.vw[c][h][r] = *reinterpret_cast<const uint32_t *>(vr + 64 * c);
            }
        }
    };
    // RING: the wave's slots, 32 rows of K and 32 rows of V each
    constexpr uint32_t kSlotBytes = 64 * D;
    constexpr int kRowsPerLoad = 1024 / D, kLoadsPer16 = 16 / kRowsPerLoad, kDma = D / 16;
    lds_byte *const ring = (lds_byte *)smem + wave * (RING > 0 ? RING : 1) * kSlotBytes;
    const uint32_t ring_base = (uint32_t)(uintptr_t)ring;
    uint32_t koff = 0, voff[4] = {0, 0, 0, 0}, lane_off[kLoadsPer16];
    if constexpr (RING > 0) {
        koff = j * D + 16 * (kb ^ ring_swizzle<D>(j));
#pragma unroll
        for (int r = 0; r < 4; r++) voff[r] = (4 * kb + r) * D + 16 * ((j >> 2) ^ ring_swizzle<D>(4 * kb + r)) + 4 * (j & 3);
#pragma unroll
        for (int q = 0; q < kLoadsPer16; q++) {                     // lane's byte inside 16 rows of a block, for the q-th load of them
            const int row = q * kRowsPerLoad + lane / (D / 16), chunk = lane % (D / 16);
            lane_off[q] = row * D + 16 * (chunk ^ ring_swizzle<D>(row));
        }
    }
    const __attribute__((address_space(4))) int32_t *bt_const = (const __attribute__((address_space(4))) int32_t *)bt;   // read only while the kernel runs: scalar loads
    auto group_id = [&](int t0, int h) { return bt_const[chunk_block_of(a, min(t0 + 16 * h, last_key & ~15))]; };
    auto dma_step = [&](uint32_t slot, const int (&id)[2], int t0) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int pos = min(t0 + 16 * h, last_key & ~15);
            const uint64_t off = (uint64_t)min((uint32_t)id[h], a.max_blk) * block_bytes + (uint64_t)head_bytes + slot_of(pos) * D;
#pragma unroll
            for (int which = 0; which < 2; which++) {
                const char *base = reinterpret_cast<const char *>(which ? a.v_cache : a.k_cache) + off;
#pragma unroll
                for (int q = 0; q < kLoadsPer16; q++)
                    __builtin_amdgcn_global_load_lds((const global_byte *)(base + lane_off[q]),
                                                     (lds_byte *)(uintptr_t)(slot + (uint32_t)((which * 32 + 16 * h) * D + q * 1024)), 16, 0, 0);
            }
        }
    };
    const int n_steps = (key_end - key_begin + STEP - 1) / STEP;
    auto step_key = [&](int i) { return key_begin + STEP * (wave + W * i); };   // first key of the wave's i-th step
    const int mine = n_steps > wave ? (n_steps - wave + W - 1) / W : 0;
    int gid[RING > 0 ? RING : 1][2];
    if constexpr (RING == 0) {
#pragma unroll
        for (int f = 0; f < NF; f++)
            if (f < mine) fetch_ids(ids[f], step_key(f));
    } else {
#pragma unroll
        for (int f = 0; f < RING; f++)
#pragma unroll
            for (int h = 0; h < 2; h++) gid[f][h] = f < mine ? group_id(step_key(f), h) : 0;
    }

    // columns of this lane and their queries: k-slots of product st are dims 64 (st / 2) + 16 kb + 8 (st % 2) + {0..7}
    int64_t item[NB];
    int last[NB];
    half8_t qf[BF8 ? 1 : NB][BF8 ? 1 : STEPS];
    long qf8[BF8 ? NB : 1][BF8 ? STEPS : 1];
    u32x2 qw[NB][STEPS];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const int c = min(t.col0 + 16 * b + j, t.cols - 1), r = chunk_row_of(a, c);
        item[b] = (int64_t)(t.row0 + r) * a.n_q_heads + kvh * a.group + (c - r * a.group);
        last[b] = a.causal ? t.p0 + r : t.ctx - 1;
#pragma unroll
        for (int st = 0; st < STEPS; st++)
            qw[b][st] = *reinterpret_cast<const u32x2 *>(a.q + item[b] * DW + 16 * (st / 2) + 4 * kb + 2 * (st % 2));
    }
    int next_id[2] = {0, 0};
    if constexpr (RING == 0) {
#pragma unroll
        for (int f = 0; f < NF; f++)
            if (f < mine) {
                load_step(steps[f], ids[f], step_key(f));
                if (f + NF < mine) fetch_ids(ids[f], step_key(f + NF));
            }
    } else {
#pragma unroll
        for (int f = 0; f < RING; f++)
            if (f < mine) dma_step(ring_base + f * kSlotBytes, gid[f], step_key(f));
#pragma unroll
        for (int h = 0; h < 2; h++)
            if (RING < mine) next_id[h] = group_id(step_key(RING), h);
    }
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
        for (int st = 0; st < STEPS; st++) {
            if constexpr (BF8) qf8[b][st] = __builtin_bit_cast(long, qw[b][st]);
            else qf[b][st] = chunk_dec8<MODE>(qw[b][st].x, qw[b][st].y);
        }
    const int tile_first = a.causal ? t.p0 + chunk_row_of(a, t.col0) : t.ctx - 1;

    float4_t o[NB][RB][4];
    float m_run[NB], mc_run[NB], l_run[NB];   // reference point (raw, and as chunk_reference gives it), the lane's share of the sum
#pragma unroll
    for (int b = 0; b < NB; b++) {
        m_run[b] = mc_run[b] = -INFINITY;
        l_run[b] = 0.f;
#pragma unroll
        for (int rb = 0; rb < RB; rb++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[b][rb][c] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    auto compute_step = [&](Step &S, int t0) {
        const bool masked = t0 + STEP - 1 > min(tile_first, last_key);   // some column does not see some key (wave-uniform)
        bool nf = false;
        if (BF8 && masked) {   // codes of inf and NaN must not meet the zero P of a column that does not see them
            uint32_t any = 0;
#pragma unroll
            for (int c = 0; c < RB; c++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t m = chunk_nonfinite(S.vw[c][h][r]);
                        S.vw[c][h][r] &= ~m;
                        any |= m;
                    }
            nf = __builtin_amdgcn_ballot_w64(any != 0) != 0;
        }
        half8_t p[NB];
        float4_t sc[NB][2];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int c = 0; c < RB; c++) {   // a key is decoded once for all column blocks
                const float4_t zero = {0.f, 0.f, 0.f, 0.f};
                if constexpr (BF8) {
                    const long k0 = __builtin_bit_cast(long, u32x2{S.kw[h][c].x, S.kw[h][c].y}), k1 = __builtin_bit_cast(long, u32x2{S.kw[h][c].z, S.kw[h][c].w});
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        sc[b][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf8_bf8(k0, qf8[b][2 * c], c == 0 ? zero : sc[b][h], 0, 0, 0);
                        sc[b][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf8_bf8(k1, qf8[b][2 * c + 1], sc[b][h], 0, 0, 0);
                    }
                } else {
                    const half8_t k0 = chunk_dec8<MODE>(S.kw[h][c].x, S.kw[h][c].y), k1 = chunk_dec8<MODE>(S.kw[h][c].z, S.kw[h][c].w);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        sc[b][h] = chunk_mfma16(k0, qf[b][2 * c], c == 0 ? zero : sc[b][h]);
                        sc[b][h] = chunk_mfma16(k1, qf[b][2 * c + 1], sc[b][h]);
                    }
                }
            }
        if (masked) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                int rel = min(last[b], last_key) - t0 - 4 * kb;         // key 16 h + 4 kb + r is hidden if 16 h + r > rel
                asm volatile("" : "+v"(rel));
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (16 * h + r > rel) sc[b][h][r] = -INFINITY;
                asm volatile("" : "+v"(sc[b][0]), "+v"(sc[b][1]));      // keeps the compares inside this rarely taken branch
            }
        }
        // P against the column's current reference point; the lane's share of the sum, needed anyway, tells whether that
        // was safe (see kGuard).  If not -- the first keys of a column, whose reference is -inf, or a score far above it --
        // the references are raised to the true maxima, the accumulators rescaled and P computed again.
        float sum[NB];
        auto exp_block = [&](auto far_c, int b, float ref) {
            constexpr bool FAR = decltype(far_c)::value;
            uint32_t pw[4];
            sum[b] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float e0 = chunk_exp<FAR>(sc[b][i >> 1][2 * (i & 1)], a.scale_log2e, ref);
                const float e1 = chunk_exp<FAR>(sc[b][i >> 1][2 * (i & 1) + 1], a.scale_log2e, ref);
                pw[i] = as_u32(__builtin_convertvector(float2p_t{e0, e1}, half2_t));
                sum[b] = dot2(pw[i], 0x3c003c00u, sum[b]);              // the sum takes the rounded values that multiply V
            }
            p[b] = __builtin_bit_cast(half8_t, u32x4{pw[0], pw[1], pw[2], pw[3]});
        };
        bool safe = true;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            exp_block(std::false_type{}, b, mc_run[b]);
            safe = safe && sum[b] < kGuard;
        }
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(!safe) != 0, 0)) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float4_t (&s)[2] = sc[b];
                float mx = max3_raw(max3_raw(s[0][0], s[0][1], s[0][2]), s[0][3], s[1][0]);
                mx = max_raw(max3_raw(mx, s[1][1], s[1][2]), s[1][3]);
                mx = max_xor32(max_xor16(mx));
                const float m_old = m_run[b], m_new = max_raw(m_old, mx);
                // a column that has seen no key keeps the reference -inf: its scores are -inf here, its P zero
                const float alpha = m_old == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_old - m_new) * a.scale_log2e);
                const float mc = chunk_reference(m_new, a.scale_log2e);
                const bool far = m_new != -INFINITY && __builtin_fabsf(mc) > kFar;
                m_run[b] = m_new;
                mc_run[b] = far ? -INFINITY : mc;                       // (-inf: such a column comes here with every step)
                l_run[b] *= alpha;
#pragma unroll
                for (int rb = 0; rb < RB; rb++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[b][rb][c] *= alpha;
                if (__builtin_amdgcn_ballot_w64(far) != 0) exp_block(std::true_type{}, b, m_new == -INFINITY ? 0.f : m_new);
                else exp_block(std::false_type{}, b, m_new == -INFINITY ? 0.f : mc);
            }
        }
#pragma unroll
        for (int b = 0; b < NB; b++) l_run[b] += sum[b];
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
            uint32_t pr[4][4];   // [pair of keys][byte]
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    const uint32_t wa = S.vw[rb][h][2 * q], wb = S.vw[rb][h][2 * q + 1];
                    uint32_t *out = pr[2 * h + q];
                    if constexpr (BF8) {
#pragma unroll
                        for (int c = 0; c < 4; c++) out[c] = perm(wb, wa, 0x000c000cu | ((uint32_t)c << 8) | ((uint32_t)(4 + c) << 24));
                    } else {   // codes of the two keys interleaved first: the decoder's pairs are then the key pairs
                        dec_word<MODE>(perm(wb, wa, 0x05010400u), out[0], out[1]);
                        dec_word<MODE>(perm(wb, wa, 0x07030602u), out[2], out[3]);
                    }
                }
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const half8_t vf = __builtin_bit_cast(half8_t, u32x4{pr[0][c], pr[1][c], pr[2][c], pr[3][c]});
#pragma unroll
                for (int b = 0; b < NB; b++) o[b][rb][c] = chunk_mfma16(vf, p[b], o[b][rb][c]);
            }
        }
        if (BF8 && nf) {   // rare: what the zeros stand for, added for the columns that see the key
            for (int key = t0; key <= min(t0 + STEP - 1, last_key); key++) {
                const uint32_t *vr = reinterpret_cast<const uint32_t *>(row_at(a.v_cache, bt[chunk_block_of(a, key)], key, 16 * kb));
#pragma unroll
                for (int rb = 0; rb < RB; rb++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t w = vr[16 * rb + r], m = chunk_nonfinite(w);
                        if (m != 0)
#pragma unroll
                            for (int c = 0; c < 4; c++)
                                if ((m >> (8 * c)) & 1u) {
                                    const float x = (float)__builtin_bit_cast(_Float16, (uint16_t)((w >> (8 * c)) << 8));
#pragma unroll
                                    for (int b = 0; b < NB; b++)
                                        if (key <= last[b]) o[b][rb][c][r] += x;
                                }
                    }
            }
        }
    };
    if constexpr (RING == 0) {
        for (int i = 0; i < mine; i += NF) {
#pragma unroll
            for (int f = 0; f < NF; f++) {
                if (i + f < mine) {
                    compute_step(steps[f], step_key(i + f));
                    if (i + f + NF < mine) {
                        load_step(steps[f], ids[f], step_key(i + f + NF));
                        if (i + f + 2 * NF < mine) fetch_ids(ids[f], step_key(i + f + 2 * NF));
                    }
                }
            }
        }
    } else {
        uint32_t slot = ring_base;
        for (int i = 0; i < mine; i++) {
            // the step's loads are older than those of the RING - 1 steps behind it, kDma loads each; at the end of the
            // range there are fewer behind it and the wave waits for all
            if (i + RING - 1 < mine) asm volatile("s_waitcnt vmcnt(%0)" :: "n"((RING - 1) * kDma) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            ring_read<D>(slot, koff, voff, steps[0]);                // complete when it returns: the slot is free again
            if (i + RING < mine) {
                dma_step(slot, next_id, step_key(i + RING));
                if (i + RING + 1 < mine) {
                    next_id[0] = group_id(step_key(i + RING + 1), 0);
                    next_id[1] = group_id(step_key(i + RING + 1), 1);
                }
            }
            compute_step(steps[0], step_key(i));
            slot = slot + kSlotBytes == ring_base + RING * kSlotBytes ? ring_base : slot + kSlotBytes;
        }
        __syncthreads();                                             // the rings become the exchange area
    }

    // ---- join the four waves: all partial results go to LDS, then W / NB waves finish a column block, a share of its
    // dims each
#pragma unroll
    for (int b = 0; b < NB; b++) {
        float l = l_run[b];
        l += __shfl_xor(l, 16, kWave);
        l += __shfl_xor(l, 32, kWave);
        if (kb == 0) {
            ml_lds[b][wave][0][j] = m_run[b];
            ml_lds[b][wave][1][j] = l;
        }
#pragma unroll
        for (int rb = 0; rb < RB; rb++)
#pragma unroll
            for (int r = 0; r < 4; r++)   // (rb, r): words 16 rb + 4 kb + r of the column
                x_lds[((b * W + wave) * RB * 4 + rb * 4 + r) * 64 + lane] = float4_t{o[b][rb][0][r], o[b][rb][1][r], o[b][rb][2][r], o[b][rb][3][r]};
    }
    __syncthreads();
    constexpr int SHARES = W / NB, UNITS = RB * 4 / SHARES;
    const int b = wave / SHARES, u0 = (wave % SHARES) * UNITS;
    const int col = t.col0 + 16 * b + j;
    if (col < t.cols) {
    float m = -INFINITY, wgt[W], sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; w++) m = fmaxf(m, ml_lds[b][w][0][j]);
#pragma unroll
    for (int w = 0; w < W; w++) {
        const float mw = ml_lds[b][w][0][j];
        wgt[w] = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - m) * a.scale_log2e);
        sum += wgt[w] * ml_lds[b][w][1][j];
    }
    const int row = chunk_row_of(a, col);
    const int64_t it = (int64_t)(t.row0 + row) * a.n_q_heads + kvh * a.group + (col - row * a.group);
    const int64_t items = narrow_items(a), at = zr * items + narrow_item(a, it, t.seq, t.row0);
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;                 // no visible key: a zero result
#pragma unroll
    for (int i = 0; i < UNITS; i++) {
        const int u = u0 + i;
        float4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; w++)
            if (wgt[w] != 0.f) x += x_lds[((b * W + w) * RB * 4 + u) * 64 + lane] * wgt[w];
        const int w4 = 16 * (u >> 2) + 4 * kb + (u & 3);
        if (a.z_narrow > 1) *reinterpret_cast<float4_t *>(a.part_narrow + at * D + 4 * w4) = x;
        else chunk_store<D, MODE>(a, it, w4, sum == 0.f ? float4_t{0.f, 0.f, 0.f, 0.f} : x * inv);
    }
    if (a.z_narrow > 1 && u0 == 0 && kb == 0) *reinterpret_cast<float2p_t *>(a.part_narrow + a.z_narrow * items * D + at * 2) = float2p_t{m, sum};
    }
    if (t.cols > a.narrow_tiles * QT) __syncthreads();               // the next tile writes the exchange area
    }
}

// ---- kernels: the LDS kernel alone, the narrow one alone, or both in one grid ------------------------------------------
// Workgroup of the LDS kernels per head dim: columns, waves, keys per tile, and waves per SIMD that the registers are for.
// The others measured (us, kernel alone; "2048 rows" is the chunk of the table at the top):
//   d = 64:  256 columns, 4 waves 142; 256 in 8 waves 176; 512 in 8 waves 171 (2048 rows, E5M2)
//   d = 128: 128 columns, 4 waves 243; 256 in 8 waves 231 + 18 of the merge that it then needs; 256 in 4 waves 258 (2048 rows, E5M2)
//   d = 256: 128 columns, 8 waves 210 / 217; 128 in 4 waves 289 / 326; 256 in 8 waves 380 / 628, spills; tiles of 32 keys 233 /
//            236; 64 columns in 4 waves, 32 keys, two workgroups per CU 285 / 300 (2048 rows, E5M2 / E4M3)
//   d = 512: 128 columns, 8 waves 425 / 543; 64 in 4 waves 901 / 1067; 128 in 4 waves 590 / 1465 (2048 rows, E5M2 / E4M3);
//            3 x 150 rows over 1501 keys, E4M3: 85 with 128 columns, 85 with 64
struct WideShape { int columns, waves, keys, occ; };
constexpr int kMost32 = 128;             // largest head dim on the 32x32 instructions
static constexpr WideShape wide_shape(int64_t d) {
    return d == 64 ? WideShape{256, 4, 64, 2} : (d == 128 ? WideShape{128, 4, 64, 2} : (d == 256 ? WideShape{128, 8, 64, 1} : WideShape{128, 8, 32, 1}));
}
// Steps in the ring of a wave of the narrow kernel: what 160 KB of LDS hold with the workgroups that the registers allow
// (0: the rows go through registers; at d = 512 one step of four waves is 128 KB, and none would be in flight behind it).
static constexpr int ring_steps(int d, int nb) { return d == 64 ? 4 : (d <= 256 ? 2 : 0); }

// 16-column blocks of the narrow kernel beside the LDS kernel.  Single rows need one (16 of them beside a chunk of 512
// rows, d = 128: 40.5 us instead of 43.8); drafts beside a prompt need two, and would be mostly empty LDS tiles with one.
constexpr int mixed_blocks(int d) { return d <= 256 ? 2 : 1; }
// Tiles of a sequence there (d = 64, 128: one grid with the LDS kernel, whose tiles would be mostly empty for drafts; the
// second ones come last in it and mostly end at once).  16 sequences of 4000 keys beside a chunk of 512 rows: 10 rows of 4
// heads, d = 128, E5M2 117 us with one tile (such sequences are the LDS kernel's then), 66 with two; 5 rows of 8 heads,
// d = 64, E4M3 42 and 37; d = 256, two launches, 63 and 66.
constexpr int mixed_tiles(int d) { return d <= 128 ? 2 : 1; }
constexpr size_t wide_lds(int d, int mode) {   // two (K, V^T) buffers; K rows of d bytes (E5M2) or halfs, 16 bytes more each
    const WideShape w = wide_shape(d);
    return (size_t)(w.keys * (mode == FEATHER_E5M2 ? d + 16 : 2 * d + 16) + 2 * d * w.keys) * 2;
}
constexpr size_t narrow_lds(int d, int nb, int ring) {   // the rings, or the exchange at the end
    const size_t join = (size_t)nb * d * 256, rings = (size_t)4 * ring * 64 * d;
    return join > rings ? join : rings;
}

template <int D, int MODE, bool PAGE16, bool ZS>
__device__ __forceinline__ void chunk_wide_body(const ChunkArgs &a, int bid) {
    constexpr WideShape w = wide_shape(D);
    if constexpr (D <= kMost32) chunk_attn32_body<D, MODE, w.columns / (32 * w.waves), w.waves, PAGE16, ZS>(a, bid);
    else chunk_attn_body<D, MODE, w.columns / (16 * w.waves), w.keys, w.waves, PAGE16, ZS>(a, bid);
}

template <int D, int MODE, bool PAGE16, bool ZS>
__global__ __launch_bounds__(64 * wide_shape(D).waves, wide_shape(D).occ) void chunk_wide_kernel(ChunkArgs a, int n_slots) {
    const int work = n_slots * a.n_kv_heads * (ZS ? a.z_wide : 1), bid = blockIdx.x;
    if (bid < work) chunk_wide_body<D, MODE, PAGE16, ZS>(a, bid);
    else chunk_fill_outside<D>(a, bid - work, gridDim.x - work, 64 * wide_shape(D).waves);
}

template <int D, int MODE, int NB, int RING>
__global__ __launch_bounds__(256, (D / 64) * NB <= 4 ? 2 : 1) void chunk_narrow_kernel(ChunkArgs a, int fill) {
    if (fill && blockIdx.y == 0) chunk_fill_outside<D>(a, blockIdx.x, gridDim.x, 256);
    const int pairs = a.n_seq * a.n_kv_heads, tile = pairs > 0 ? blockIdx.x / pairs : 0;
    if (a.n_seq > 0) chunk_narrow_body<D, MODE, NB, RING>(a, blockIdx.x - tile * pairs, tile, blockIdx.y);
}

// A batch of long and short runs of rows: the tiles first, whose matrix work then shares the CUs with the streaming of the
// short ones' caches (one after the other they leave the memory and the matrix cores idle in turn).
template <int D, int MODE, bool PAGE16, bool ZS>
__global__ __launch_bounds__(256, wide_shape(D).occ) void chunk_mixed_kernel(ChunkArgs a, int n_slots) {
    constexpr int NB = mixed_blocks(D);
    int bid = blockIdx.x;
    const int wide = n_slots * a.n_kv_heads * (ZS ? a.z_wide : 1), pairs = a.n_seq * a.n_kv_heads, ranges = pairs * a.z_narrow, narrow = ranges * a.narrow_tiles;
    if (bid < wide) {
        chunk_wide_body<D, MODE, PAGE16, ZS>(a, bid);
        return;
    }
    bid -= wide;
    if (bid < narrow) {
        const int tile = bid / ranges, at = bid - tile * ranges, zr = at / pairs;
        chunk_narrow_body<D, MODE, NB, PAGE16 ? ring_steps(D, NB) : 0>(a, at - zr * pairs, tile, zr);
    } else {
        chunk_fill_outside<D>(a, bid - narrow, gridDim.x - wide - narrow, 256);
    }
}

// Adds the key ranges of a column in range order.  A workgroup holds 256 / (DW * zl) items (row, head); an item's dims
// lie along DW threads, and zl of these rows of threads take the item's ranges in turn and are joined through LDS, so
// that few items of many ranges are not one long chain of loads.  Rows of no sequence are zeroed here (fill) or left
// alone; rows whose kernel had a single range have their result already.
// chunk_plan makes ranges to fill kWideGroups workgroups of the LDS kernel, or up to 3 kCus of the narrow one, with two ranges
// or more per sequence: a call with ranges has few sequences.  Their offsets are kept in LDS, so the search for a row's sequence
// is no chain of loads.
constexpr int kWideGroups = 512, kCus = 256, kMergeSeqs = 512;
static_assert(kWideGroups / 2 <= kMergeSeqs && 3 * kCus / 2 <= kMergeSeqs, "offsets of more sequences than the merge keeps");

template <int D, int MODE>
__global__ __launch_bounds__(256) void chunk_merge_kernel(ChunkArgs a, int qt_wide_log2, int bn_wide, int qt_narrow_log2, int zl_log2) {
    constexpr int DW = D / 4, G = 4;
    __shared__ float4_t x_lds[256];
    __shared__ float2p_t ml_lds[256];
    __shared__ int cu_lds[kMergeSeqs + 1];
    for (int s = threadIdx.x; s <= a.n_seq; s += 256) cu_lds[s] = chunk_clamp_row(a.cu_seqlens[s], a.total_rows);
    __syncthreads();
    const int tid = threadIdx.x, zl = 1 << zl_log2, w4 = tid % DW, zi = (tid / DW) & (zl - 1);
    const int items = a.total_rows * a.n_q_heads;           // below 2^30
    const int item = (int)blockIdx.x * ((256 / DW) >> zl_log2) + ((tid / DW) >> zl_log2);
    int used = 0;
    bool zero = false;
    const float *part = a.part;                        // partial results of the row's kernel: [range][item][D], [range][item] pairs
    int64_t part_items = items, part_item = item;
    int z = 1;
    if (item < items) {
        const int row = (int)(__umulhi(2u * (uint32_t)item, a.head_mul) >> a.head_shift), head = item - row * a.n_q_heads;
        int lo = 0, hi = a.n_seq;                      // last sequence that starts at or before the row
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (cu_lds[mid] <= row) lo = mid; else hi = mid;
        }
        const int r0 = cu_lds[lo], r1 = max(cu_lds[lo + 1], r0);
        if (row < r0 || row >= r1) {
            zero = a.fill;
        } else {
            const int ctx = min(max(a.ctx_lens[lo], 0), a.max_blocks * a.block_size), p0 = ctx - (r1 - r0);
            const int cols = (r1 - r0) * a.group;
            const bool narrow = cols <= a.col_split;
            const int qt_log2 = narrow ? qt_narrow_log2 : qt_wide_log2;
            z = narrow ? a.z_narrow : a.z_wide;
            const int col = (row - r0) * a.group + head - chunk_row_of(a, head) * a.group, col_end = ((col >> qt_log2) + 1) << qt_log2;   // of its tile
            const int keys = a.causal ? max(p0 + chunk_row_of(a, min(col_end, cols) - 1) + 1, 0) : ctx;
            if (z > 1) {
                if (narrow) {
                    part = a.part_narrow;
                    part_items = narrow_items(a);
                    part_item = narrow_item(a, item, lo, r0);
                }
                const int per = narrow ? chunk_range_keys(keys, z, kNarrowStep, *reinterpret_cast<const int *>(part + part_items * z * (D + 2)))
                                       : chunk_range_keys(keys, z, bn_wide, kChunkMinKeys);
                used = (keys + per - 1) / per;
                zero = used == 0;
            }
        }
    }
    const float2p_t *ml = reinterpret_cast<const float2p_t *>(part + z * part_items * D);
    // A range without a maximum has only hidden keys (sum and accumulators are zero) or only NaN scores (then they are NaN,
    // and so is the row): its weight is zero, which keeps a NaN, and it is not left out.
    auto weight = [&](float m_range, float m_all) { return m_range == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_range - m_all) * a.scale_log2e); };
    float m = -INFINITY, l = 0.f;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int z0 = zi; z0 < used; z0 += G * zl) {       // G ranges per turn, all loads before the first use
        float2p_t x[G];
        float4_t y[G];
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int64_t at = min(z0 + g * zl, used - 1) * part_items + part_item;
            x[g] = ml[at];
            y[g] = *reinterpret_cast<const float4_t *>(part + at * D + 4 * w4);
        }
        float mg = m;
#pragma unroll
        for (int g = 0; g < G; g++) {
            if (z0 + g * zl >= used) x[g] = float2p_t{-INFINITY, 0.f};
            mg = fmaxf(mg, x[g][0]);
        }
        const float keep = weight(m, mg);
        l *= keep;
        acc *= keep;
#pragma unroll
        for (int g = 0; g < G; g++) {
            if (z0 + g * zl >= used) continue;
            const float w = weight(x[g][0], mg);
            l += x[g][1] * w;
            acc += y[g] * w;
        }
        m = mg;
    }
    if (zl > 1) {
        x_lds[tid] = acc;
        ml_lds[tid] = float2p_t{m, l};
        __syncthreads();
        if (zi > 0) return;
        float mg = m;
        for (int k = 1; k < zl; k++) mg = fmaxf(mg, ml_lds[tid + k * DW][0]);
        const float keep = weight(m, mg);
        l *= keep;
        acc *= keep;
        for (int k = 1; k < zl; k++) {
            const float2p_t x = ml_lds[tid + k * DW];
            const float w = weight(x[0], mg);
            l += x[1] * w;
            acc += x_lds[tid + k * DW] * w;
        }
    }
    if (used > 0 || zero) chunk_store<D, MODE>(a, item, w4, l == 0.f ? float4_t{0.f, 0.f, 0.f, 0.f} : acc * (1.0f / l));
}

// ---- host ---------------------------------------------------------------------------------------------------------

// How a call is cut: which kernels run, their tiles, and into how many key ranges.
struct ChunkPlan {
    bool wide, narrow;
    int nb, tiles;          // 16-column blocks of a narrow tile; tiles of a sequence
    int col_split;
    int z_wide, z_narrow, narrow_rows;
    float per_group;
    int64_t wide_bytes, narrow_bytes;   // of the workspace, per range
};

static int log2_of(int64_t x) { int l = 0; while ((1ll << l) < x) l++; return l; }

static int wide_columns(int64_t d) { return wide_shape(d).columns; }
// Most 16-column blocks of a tile of the narrow kernel: the accumulators and queries of two waves per SIMD (one at d = 256
// and 512).  d = 128 with four blocks, one wave per SIMD: 32 sequences of 4096 keys, 64 columns, E5M2 74 us instead of 64.
static constexpr int narrow_blocks(int64_t d) { return d == 64 ? 4 : (d <= 256 ? 2 : 1); }

// Sequences of at most so many columns (in several tiles then, next to each other on an XCD) take the narrow kernel.  It
// decodes for its own wave what the LDS kernel decodes once for a workgroup, and needs neither its barriers nor as many key
// ranges.  LDS kernel against narrow kernel, us with the merge, n sequences of 4096 keys:
//   d = 64:  256 columns 100 / 68 (n = 32, E4M3), 27 / 22 (4, E5M2); 512: 150 / 130 (32, E4M3), 31 / 29 (4, E5M2); 1024: 241 / 247
//            (32, E4M3), 38 / 45 (4, E5M2)
//   d = 128: 128 columns 143 / 121 (32, E5M2), 32 / 37 (4, E4M3); 256: 249 / 271 (32, E5M2), 42 / 57 (4, E4M3)
//   d = 256: 64 columns 47 / 42 (4 of 8192, E4M3), 74 / 73 (16, E5M2); 128: 63 / 70, 95 / 70
//   d = 512: 32 columns 50 / 41 (4 of 8192, E4M3), 74 / 59 (16, E5M2); 64: 55 / 65, 85 / 135
static int narrow_columns(int64_t d) { return d == 64 ? 512 : (d == 128 ? 128 : (d == 256 ? 64 : 32)); }

static int64_t chunk_slots(int64_t total_rows, int64_t n_seq, int64_t group, int qt) { return total_rows * group / qt + n_seq; }

static int ranges_for(int64_t tiles, int64_t target, int64_t max_ctx, int64_t min_keys) {
    int64_t z = target / (tiles > 0 ? tiles : 1);
    const int64_t most = (max_ctx + min_keys - 1) / min_keys;
    if (z > most) z = most;
    if (z > 128) z = 128;
    return z < 1 ? 1 : (int)z;
}

static ChunkPlan chunk_plan(int64_t n_seq, int64_t total_rows, int64_t n_q_heads, int64_t n_kv_heads, int64_t d, int64_t max_ctx,
                            int64_t max_q_len) {
    ChunkPlan p;
    const int64_t group = n_q_heads / n_kv_heads;
    const int64_t rows_most = max_q_len > 0 && max_q_len < total_rows ? max_q_len : total_rows;   // rows of the longest sequence, if the hint is right
    const int64_t cols = rows_most * group;
    if (cols <= narrow_columns(d)) {    // all sequences are short (or the hint is wrong: more tiles each)
        p.narrow = true;
        p.wide = false;
        p.col_split = kAnyColumns;
        const int64_t apart = n_seq * n_kv_heads * ranges_for(1, 128, max_ctx, kNarrowMinKeys);   // workgroups, at most, before columns are cut
        auto tiles = [&](int nb) { return cols > 16 * nb ? (cols + 16 * nb - 1) / (16 * nb) : 1; };
        // Tiles as wide as they get read the cache once; narrow ones are more workgroups, where a short context allows no
        // ranges: two requests of 300 keys and 40 columns 9.9 us in one tile each, 6.3 in three; 32 requests of up to 4096 keys
        // 24 us with 64 columns, 29 with 32, 32 with 16.
        p.nb = 1;
        while (p.nb < narrow_blocks(d) && tiles(p.nb) > 1 && apart * tiles(p.nb) > 256) p.nb *= 2;
        p.tiles = (int)tiles(p.nb);
    } else {
        p.wide = true;
        p.nb = mixed_blocks((int)d);
        p.tiles = mixed_tiles((int)d);
        // with n_seq - 1 sequences of the longest length, can the last one be short?  (If the hint is wrong the LDS kernel
        // takes the short ones too.)
        const int64_t least = total_rows - (n_seq - 1) * rows_most;
        p.narrow = n_seq > 1 && (least < 1 ? 1 : least) * group <= 16 * p.nb * p.tiles;   // (one row has `group` columns)
        p.col_split = p.narrow ? 16 * p.nb * p.tiles : 0;
    }
    p.narrow_rows = p.wide && p.narrow ? (int)(p.col_split / group) : 0;
    const int64_t each = n_seq > 0 ? (total_rows + n_seq - 1) / n_seq * group : 1;   // columns of a sequence of average length
    // 512 workgroups, two per CU: a chunk of 2048 rows, d = 64, 142 + 11 us; 256: 198; 1024: 141 + 14.  16 single rows beside
    // 512 rows, d = 128, 136 tiles: 512 are three ranges, 43.6 + 8.2 us; 256 one, 56 + 5; 272 two, 42.1 + 7.6; 1024 seven,
    // 54 + 13.  (The workgroups of the narrow part in the same grid are not counted.)
    p.z_wide = p.wide ? ranges_for(n_seq * ((each + wide_columns(d) - 1) / wide_columns(d)) * n_kv_heads, kWideGroups, max_ctx, kChunkMinKeys) : 1;
    // the chip holds 256 workgroups of a kernel that fills a CU's registers, two or three times as many of a smaller one
    // (drafts of 32 requests, d = 64, 64 columns: 512 workgroups 24 us, 768 29, 384 28)
    const int weight = (int)(d / 64) * p.nb;
    const int64_t groups = kCus * (weight <= 2 ? 3 : (weight <= 4 ? 2 : 1));
    const int64_t tiles = (p.wide ? n_seq : n_seq * ((each + 16 * p.nb - 1) / (16 * p.nb))) * n_kv_heads;
    // twice the even share, for contexts of different lengths
    p.z_narrow = p.narrow && 2 * tiles <= groups ? ranges_for(tiles, 2 * groups, max_ctx, kNarrowMinKeys) : 1;
    p.per_group = (float)n_kv_heads / (float)(groups - tiles > 0 ? groups - tiles : 1);
    p.wide_bytes = total_rows * n_q_heads * (d + 2) * 4;
    p.narrow_bytes = (p.narrow_rows ? n_seq * p.narrow_rows : total_rows) * n_q_heads * (d + 2) * 4;
    return p;
}

static int64_t chunk_wide_scratch(const ChunkPlan &p) { return p.z_wide > 1 ? (p.z_wide * p.wide_bytes + 15) / 16 * 16 : 0; }
static int64_t chunk_narrow_scratch(const ChunkPlan &p) { return p.z_narrow > 1 ? p.z_narrow * p.narrow_bytes + 16 : 0; }

template <class Kernel>
static int launch_chunk_kernel(Kernel kern, dim3 grid, int threads, size_t lds, hipStream_t s, const ChunkArgs &a, int arg, unsigned long long &lds_raised) {
    const char *me = "feather_paged_chunk_attn_fp8";
    hipError_t e = raise_lds_limit(reinterpret_cast<const void *>(kern), lds + 4096, lds_raised);   // (and the kernels' static arrays)
    FEATHER_CHECK(e == hipSuccess, FEATHER_ELAUNCH, "%s: cannot raise LDS limit: %s", me, hipGetErrorString(e));
    hipLaunchKernelGGL(kern, grid, dim3(threads), lds, s, a, arg);
    return check_launch(me);
}

template <int D, int MODE, int NB, int RING>
static int launch_chunk_narrow(const ChunkArgs &a, bool fill, hipStream_t s) {
    const int64_t pairs = a.n_seq > 0 ? (int64_t)a.n_seq * a.n_kv_heads * a.narrow_tiles : kChunkFillGroups;
    FEATHER_CHECK(pairs * a.z_narrow < (1ll << 31), FEATHER_ESHAPE, "feather_paged_chunk_attn_fp8: grid too large");
    static unsigned long long lds_raised = 0;
    return launch_chunk_kernel(chunk_narrow_kernel<D, MODE, NB, RING>, dim3((unsigned)pairs, (unsigned)a.z_narrow), 256, narrow_lds(D, NB, RING), s, a,
                               fill ? 1 : 0, lds_raised);
}

template <int D, int MODE, bool PAGE16, bool ZS>
static int launch_chunk_wide(const ChunkArgs &a, bool narrow, bool fill, hipStream_t s) {
    constexpr WideShape w = wide_shape(D);
    constexpr int NB = mixed_blocks(D), RING = PAGE16 ? ring_steps(D, NB) : 0;
    constexpr bool kOneGrid = w.waves == 4;            // both kernels' workgroups have four waves
    const int64_t slots = chunk_slots(a.total_rows, a.n_seq, a.group, w.columns);
    const int64_t wide = slots * a.n_kv_heads * a.z_wide, more = narrow && kOneGrid ? (int64_t)a.n_seq * a.n_kv_heads * a.narrow_tiles * a.z_narrow : 0;
    FEATHER_CHECK(wide + more + kChunkFillGroups < (1ll << 31), FEATHER_ESHAPE, "feather_paged_chunk_attn_fp8: grid too large");
    const dim3 grid((unsigned)(wide + more + (fill ? kChunkFillGroups : 0)));
    if constexpr (kOneGrid)
        if (narrow) {
            constexpr size_t lds = wide_lds(D, MODE) > narrow_lds(D, NB, RING) ? wide_lds(D, MODE) : narrow_lds(D, NB, RING);
            static unsigned long long lds_raised = 0;
            return launch_chunk_kernel(chunk_mixed_kernel<D, MODE, PAGE16, ZS>, grid, 256, lds, s, a, (int)slots, lds_raised);
        }
    static unsigned long long lds_raised = 0;
    const int rc = launch_chunk_kernel(chunk_wide_kernel<D, MODE, PAGE16, ZS>, grid, 64 * w.waves, wide_lds(D, MODE), s, a, (int)slots, lds_raised);
    if (rc != FEATHER_OK || !narrow) return rc;
    return launch_chunk_narrow<D, MODE, NB, RING>(a, false, s);
}

template <int D, int MODE, bool PAGE16>
static int launch_chunk(const ChunkArgs &a, const ChunkPlan &p, hipStream_t s) {
    const bool merge = a.z_wide > 1 || a.z_narrow > 1;
    const bool fill = a.fill && !merge;                      // rows outside every sequence: the merge's work, or the first kernel's
    int rc = FEATHER_OK;
    if (p.wide) {
        rc = a.z_wide > 1 ? launch_chunk_wide<D, MODE, PAGE16, true>(a, p.narrow, fill, s) : launch_chunk_wide<D, MODE, PAGE16, false>(a, p.narrow, fill, s);
    } else {
        if (p.nb == 1) rc = launch_chunk_narrow<D, MODE, 1, PAGE16 ? ring_steps(D, 1) : 0>(a, fill, s);
        if constexpr (D <= 256)
            if (p.nb == 2) rc = launch_chunk_narrow<D, MODE, 2, PAGE16 ? ring_steps(D, 2) : 0>(a, fill, s);
        if constexpr (D == 64)
            if (p.nb == 4) rc = launch_chunk_narrow<D, MODE, 4, PAGE16 ? ring_steps(D, 4) : 0>(a, fill, s);
    }
    if (rc != FEATHER_OK || !merge) return rc;
    constexpr int DW = D / 4;
    int zl = 0;                                              // four ranges per thread and turn; rows of the LDS kernel have few
    while (!p.wide && (4 << zl) < a.z_narrow && (DW << zl) < 256) zl++;
    const int64_t per_group = (256 / DW) >> zl, items = (int64_t)a.total_rows * a.n_q_heads;
    hipLaunchKernelGGL((chunk_merge_kernel<D, MODE>), dim3((unsigned)((items + per_group - 1) / per_group)), dim3(256), 0, s, a,
                       log2_of(wide_columns(D)), wide_shape(D).keys, log2_of(16 * p.nb), zl);
    return check_launch("feather_paged_chunk_attn_fp8 (merge of the key ranges)");
}

template <int MODE, bool PAGE16>
static int dispatch_chunk(const ChunkArgs &a, const ChunkPlan &p, int64_t d, hipStream_t s) {
    switch (d) {
        case 64: return launch_chunk<64, MODE, PAGE16>(a, p, s);
        case 128: return launch_chunk<128, MODE, PAGE16>(a, p, s);
        case 256: return launch_chunk<256, MODE, PAGE16>(a, p, s);
        default: return launch_chunk<512, MODE, PAGE16>(a, p, s);
    }
}

}  // namespace feather

using namespace feather;

extern "C" int64_t feather_paged_chunk_attn_scratch_bytes(int64_t n_seq, int64_t total_rows, int64_t n_q_heads,
                                                          int64_t n_kv_heads, int64_t d, int64_t max_ctx,
                                                          int64_t max_q_len) {
    if (n_seq <= 0 || total_rows <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || d <= 0 || max_ctx <= 0 || max_q_len < 0) return 0;
    const ChunkPlan p = chunk_plan(n_seq, total_rows, n_q_heads, n_kv_heads, d, max_ctx, max_q_len);
    return chunk_wide_scratch(p) + chunk_narrow_scratch(p);
}

extern "C" int feather_paged_chunk_attn_fp8(const void *q, const void *k_cache, const void *v_cache, const void *block_tables,
                                            const void *cu_seqlens, const void *ctx_lens, void *out, int out_kind, int fill,
                                            void *scratch, int64_t scratch_bytes, int64_t n_seq, int64_t total_rows,
                                            int64_t n_q_heads, int64_t n_kv_heads, int64_t d, int64_t block_size,
                                            int64_t max_blocks, int64_t n_blocks, int64_t max_q_len, int causal, int mode,
                                            float scale, void *stream) {
    const char *me = "feather_paged_chunk_attn_fp8";
    FEATHER_CHECK(mode == FEATHER_E5M2 || mode == FEATHER_E4M3, FEATHER_EMODE, "%s: mode %d not supported", me, mode);
    FEATHER_CHECK(n_seq >= 0 && total_rows >= 0 && n_q_heads > 0 && n_kv_heads > 0 && block_size > 0 && max_blocks >= 0 &&
                      max_q_len >= 0 && scratch_bytes >= 0,
                  FEATHER_EINVAL, "%s: bad shape", me);
    FEATHER_CHECK(n_blocks >= 1 && n_blocks < (1ll << 31), FEATHER_EINVAL, "%s: n_blocks=%lld: the cache must hold at least one block",
                  me, (long long)n_blocks);
    FEATHER_CHECK(causal == 0 || causal == 1, FEATHER_EINVAL, "%s: causal must be 0 or 1", me);
    FEATHER_CHECK(fill == 0 || fill == 1, FEATHER_EINVAL, "%s: fill must be 0 or 1", me);
    FEATHER_CHECK(out_kind == FEATHER_CHUNK_OUT_F32 || out_kind == FEATHER_CHUNK_OUT_F16 || out_kind == FEATHER_CHUNK_OUT_PACKED,
                  FEATHER_EINVAL, "%s: bad output kind %d", me, out_kind);
    FEATHER_CHECK(n_q_heads % n_kv_heads == 0, FEATHER_ESHAPE, "%s: n_q_heads=%lld not a multiple of n_kv_heads=%lld", me,
                  (long long)n_q_heads, (long long)n_kv_heads);
    FEATHER_CHECK(d == 64 || d == 128 || d == 256 || d == 512, FEATHER_ESHAPE, "%s: head dim %lld not supported (64, 128, 256, 512)",
                  me, (long long)d);
    FEATHER_CHECK(scale > 0.f && scale <= 2.3e38f, FEATHER_EINVAL,          // scale * log2 e is finite too
                  "%s: scale must be positive and finite (the running maximum is kept on raw scores)", me);
    FEATHER_CHECK(block_size < (1ll << 30) && max_blocks < (1ll << 30) && max_blocks * block_size < (1ll << 30) &&
                      total_rows < (1ll << 30) && n_seq < (1ll << 30) && n_q_heads < (1ll << 20) &&
                      total_rows * n_q_heads < (1ll << 30),
                  FEATHER_ESHAPE, "%s: shape too large", me);
    FEATHER_CHECK(n_blocks * n_kv_heads < (1ll << 32) && n_blocks * n_kv_heads * block_size < (1ll << 32) &&
                      n_kv_heads * block_size * d < (1ll << 31),
                  FEATHER_ESHAPE, "%s: a cache of more than 2^32 rows, or a block of 2 GiB", me);
    if (total_rows == 0) return FEATHER_OK;
    if (n_seq == 0 && !fill) return FEATHER_OK;
    FEATHER_CHECK(q && k_cache && v_cache && out && cu_seqlens && (n_seq == 0 || (ctx_lens && (block_tables || max_blocks == 0))), FEATHER_EINVAL,
                  "%s: null pointer", me);
    FEATHER_CHECK(aligned(q, 8) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 16) && aligned(scratch, 16) &&
                      aligned(block_tables, 4) && aligned(cu_seqlens, 4) && aligned(ctx_lens, 4),
                  FEATHER_EINVAL, "%s: misaligned pointer", me);
    ChunkPlan p = chunk_plan(n_seq, total_rows, n_q_heads, n_kv_heads, d, max_blocks * block_size, max_q_len);
    const int64_t room = scratch && n_seq > 0 ? scratch_bytes : 0;   // a smaller workspace: fewer ranges
    while (chunk_wide_scratch(p) > room) p.z_wide--;
    while (chunk_wide_scratch(p) + chunk_narrow_scratch(p) > room) p.z_narrow--;
    auto divisor = [](int64_t size, uint32_t &mul, int &shift) {   // see ChunkArgs
        shift = 0;
        while ((1ll << shift) < size) shift++;
        mul = (uint32_t)((1ull << (31 + shift)) / (uint64_t)size + 1);
    };
    ChunkArgs a;
    divisor(block_size, a.div_mul, a.div_shift);
    divisor(n_q_heads / n_kv_heads, a.group_mul, a.group_shift);
    divisor(n_kv_heads, a.kv_mul, a.kv_shift);
    divisor(n_q_heads, a.head_mul, a.head_shift);
    a.q = (const uint32_t *)q; a.k_cache = (const uint32_t *)k_cache; a.v_cache = (const uint32_t *)v_cache;
    a.block_tables = (const int32_t *)block_tables; a.cu_seqlens = (const int32_t *)cu_seqlens; a.ctx_lens = (const int32_t *)ctx_lens;
    a.out = out; a.part = (float *)scratch;
    a.n_seq = (int)n_seq; a.total_rows = (int)total_rows; a.n_q_heads = (int)n_q_heads; a.n_kv_heads = (int)n_kv_heads;
    a.group = (int)(n_q_heads / n_kv_heads); a.block_size = (int)block_size; a.max_blocks = (int)max_blocks;
    a.max_blk = (uint32_t)(n_blocks - 1);
    a.causal = causal; a.out_kind = out_kind; a.fill = fill;
    a.z_wide = p.z_wide; a.z_narrow = p.z_narrow; a.per_group = p.per_group; a.narrow_rows = p.narrow_rows; a.narrow_tiles = p.tiles;
    a.part_narrow = reinterpret_cast<float *>(static_cast<char *>(scratch) + chunk_wide_scratch(p)); a.col_split = p.col_split;
    a.scale_log2e = scale * 1.4426950408889634f;
    a.shift_raw = std::fmin(kShift / a.scale_log2e, 1.0e38f);          // (finite for a subnormal scale too)
    a.raise_raw = std::fmin((kShift + kLazy) / a.scale_log2e, 3.0e38f);
    hipStream_t s = (hipStream_t)stream;
    const bool al = block_size % 16 == 0;
    if (mode == FEATHER_E5M2) return al ? dispatch_chunk<FEATHER_E5M2, true>(a, p, d, s) : dispatch_chunk<FEATHER_E5M2, false>(a, p, d, s);
    return al ? dispatch_chunk<FEATHER_E4M3, true>(a, p, d, s) : dispatch_chunk<FEATHER_E4M3, false>(a, p, d, s);
}
