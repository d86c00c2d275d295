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
// rate, and the error (2^-11 / sqrt(3) of each P, random in sign) is of the size of the fp16 result's own rounding.
// The denominator sums the rounded P.
#include <type_traits>

#include "common.h"

namespace feather {

typedef float float2p_t __attribute__((ext_vector_type(2)));

enum ChunkOut { kChunkF32 = 0, kChunkF16 = 1, kChunkPacked = 2 };

struct ChunkArgs {
    const uint32_t *q, *k_cache, *v_cache;
    const int32_t *block_tables, *cu_seqlens, *ctx_lens;
    void *out;
    float *part;            // partial results of the key ranges (z > 1)
    int n_seq, total_rows, n_q_heads, n_kv_heads, group, block_size, max_blocks;
    uint32_t max_blk;       // last block of the cache: an entry outside the cache is read as this one
    uint32_t div_mul;       // pos / block_size = umulhi(2 pos, div_mul) >> div_shift for 0 <= pos < 2^31
    int div_shift;
    int causal, z, out_kind, fill;
    float scale_log2e;
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

__device__ __forceinline__ bool chunk_find_tile(const ChunkArgs &a, int slot, int qt, ChunkTile &t) {
    const int lane = lane_id();
    int below = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += kWave) {
        const int s = s0 + lane;
        const bool hit = s < a.n_seq &&
                         (int64_t)chunk_clamp_row(a.cu_seqlens[min(s, a.n_seq - 1)], a.total_rows) * a.group / qt + s <= slot;
        const uint64_t m = __builtin_amdgcn_ballot_w64(hit);
        below += __builtin_popcountll(m);
        if (m != ~0ull) break;
    }
    if (below == 0) return false;
    t.seq = __builtin_amdgcn_readfirstlane(below - 1);
    t.row0 = chunk_clamp_row(a.cu_seqlens[t.seq], a.total_rows);
    t.rows = max(chunk_clamp_row(a.cu_seqlens[t.seq + 1], a.total_rows) - t.row0, 0);
    t.cols = t.rows * a.group;
    const int n_tiles = (t.cols + qt - 1) / qt;
    const int tile = slot - (int)((int64_t)t.row0 * a.group / qt + t.seq);
    if (tile < 0 || tile >= n_tiles) return false;
    // causal: the tiles with the longest key loops start first
    t.col0 = (a.causal ? n_tiles - 1 - tile : tile) * qt;
    t.ctx = min(max(a.ctx_lens[t.seq], 0), a.max_blocks * a.block_size);
    t.p0 = t.ctx - t.rows;
    t.keys = a.causal ? max(t.p0 + (min(t.col0 + qt, t.cols) - 1) / a.group + 1, 0) : t.ctx;
    return true;
}

// Keys per range of a tile that can see `keys` keys, when up to z workgroups share it.
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
    if (a.out_kind == kChunkF32) {
        *reinterpret_cast<float4_t *>(static_cast<float *>(a.out) + item * D + 4 * w4) = x;
    } else if (a.out_kind == kChunkF16) {
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
    const int words = a.out_kind == kChunkF32 ? 4 : (a.out_kind == kChunkF16 ? 2 : 1);
    uint32_t *out = static_cast<uint32_t *>(a.out);
    for (int64_t i = (int64_t)part * threads + threadIdx.x; i < (first + (int64_t)(a.total_rows - last)) * unit * words;
         i += (int64_t)parts * threads) {
        const int64_t at = i < first * unit * words ? i : i + (int64_t)(last - first) * unit * words;
        out[at] = 0u;
    }
}

constexpr int kChunkFillGroups = 8;    // workgroups of a grid that only look after rows outside every sequence
constexpr int kChunkMinKeys = 256;     // a key range is not cut below this

// ---- tiles through LDS --------------------------------------------------------------------------------------------
// One workgroup (WAVES waves) owns 16 * QB * WAVES columns, each wave 16 * QB of them for the whole key loop.  Tiles
// of BN keys are fetched packed through the block table into registers two tiles ahead (their block ids three tiles
// ahead: a table entry is never waited for), decoded into the other LDS buffer one tile ahead, and read by all waves.
// ALIGN4: block_size % 4 == 0, so four keys from a multiple of four on share a block (one table lookup).
template <int D, int MODE, int QB, int BN, int OCC, int WAVES, bool ALIGN4, bool ZS>
__global__ __launch_bounds__(64 * WAVES, OCC) void chunk_attn_kernel(ChunkArgs a, int n_slots, int col_min) {
    constexpr int DW = D / 4;
    constexpr bool BF8 = MODE == FEATHER_E5M2;
    constexpr int KS = BF8 ? (D + 16) / 2 : D + 8;   // K row pitch in LDS, in fp16 units (bf8: D + 16 bytes)
    constexpr int VS = BN, CH = BN / 8;
    constexpr int kThreads = 64 * WAVES, QT = 16 * QB * WAVES;
    constexpr int UNITS = BN * D / 16;
    constexpr int NU = UNITS >= kThreads ? UNITS / kThreads : 1;
    constexpr bool ALL_STAGE = UNITS >= kThreads;
    static_assert(UNITS % 64 == 0 && (ALL_STAGE ? UNITS % kThreads == 0 : true), "tile / workgroup mismatch");
    constexpr int DB = D / 16, STEPS = D / 32, KB16 = BN / 16, KB32 = BN / 32;
    constexpr int kBufHalfs = BN * KS + D * VS;

    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    _Float16 *const lds = reinterpret_cast<_Float16 *>(smem);
    auto swz = [](int row) { return (row ^ (row >> 2)) & (CH - 1); };

    const int work = n_slots * a.n_kv_heads * (ZS ? a.z : 1);
    int bid = blockIdx.x;
    if (bid >= work) {
        chunk_fill_outside<D>(a, bid - work, gridDim.x - work, kThreads);
        return;
    }
    if (work % 8 == 0) bid = (bid % 8) * (work / 8) + bid / 8;   // an XCD (own L2) works through neighbouring tiles of one KV head
    int zr = 0;
    if constexpr (ZS) {
        zr = bid % a.z;
        bid /= a.z;
    }
    const int kvh = bid / n_slots;
    ChunkTile t;
    if (!chunk_find_tile(a, bid % n_slots, QT, t)) return;
    if (t.cols < col_min) return;                      // a short sequence: the other kernel's work

    int key_begin = 0, key_end = t.keys;
    if constexpr (ZS) {
        const int per = chunk_range_keys(t.keys, a.z, BN, kChunkMinKeys);
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
        const int c = min(qc0 + 16 * b + j, t.cols - 1), r = c / a.group;
        item[b] = (int64_t)(t.row0 + r) * a.n_q_heads + kvh * a.group + (c - r * a.group);
        last[b] = a.causal ? t.p0 + r : t.ctx - 1;
    }
    const int wave_first = a.causal ? t.p0 + min(qc0, t.cols - 1) / a.group : t.ctx - 1;     // smallest and largest last key of the wave
    const int wave_last = a.causal ? t.p0 + min(qc0 + 16 * QB - 1, t.cols - 1) / a.group : t.ctx - 1;
    const int tile_first = a.causal ? t.p0 + t.col0 / a.group : t.ctx - 1;
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

    float4_t o[QB][DB + 1];          // [DB]: row sums of P, from a constant block of ones
    float m_run[QB];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        m_run[b] = -INFINITY;
#pragma unroll
        for (int d = 0; d <= DB; d++) o[b][d] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    const float lazy_raw = 8.f / a.scale_log2e;
    const _Float16 one_or_zero = (j & 3) == 0 ? (_Float16)1 : (_Float16)0;
    const half8_t ones = {one_or_zero, one_or_zero, one_or_zero, one_or_zero, one_or_zero, one_or_zero, one_or_zero, one_or_zero};

    u32x4 kreg[NU];
    uint32_t vreg[NU][4];
    int kid[NU], vid[NU][ALIGN4 ? 1 : 4];
    auto fetch_ids = [&](int key0) {
        if (!ALL_STAGE && tid >= UNITS) return;
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int u = tid + kThreads * i;
            kid[i] = bt[chunk_block_of(a, min(key0 + u / (D / 16), key_end - 1))];
#pragma unroll
            for (int r = 0; r < (ALIGN4 ? 1 : 4); r++)
                vid[i][r] = bt[chunk_block_of(a, min(key0 + 4 * (u / DW) + r, key_end - 1))];
        }
    };
    auto row_of = [&](int id, int pos) {               // cache row in 32 bits (the host checks that every row fits)
        const uint32_t slot = (uint32_t)pos - chunk_block_of(a, pos) * (uint32_t)a.block_size;
        return (int64_t)(uint32_t)(min((uint32_t)id, a.max_blk) * (uint32_t)block_rows + (uint32_t)head_rows + slot);
    };
    auto prefetch = [&](int key0) {                    // the ids of this tile are in kid / vid
        if (!ALL_STAGE && tid >= UNITS) return;
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int u = tid + kThreads * i;
            const int kp = key0 + u / (D / 16), c16 = u % (D / 16);
            kreg[i] = u32x4{0, 0, 0, 0};
            if (kp < key_end) kreg[i] = *reinterpret_cast<const u32x4 *>(a.k_cache + row_of(kid[i], kp) * DW + 4 * c16);
            const int ddw = u % DW, vp = key0 + 4 * (u / DW);
            if constexpr (ALIGN4) {
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
        if (!ALL_STAGE && tid >= UNITS) return 0;
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
    if (BF8 && a.causal) nf = __syncthreads_or(nf);
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
                // The reference point is raised only when a column exceeds it by 2^8 (O / l does not depend on it).  A
                // column that has seen no key yet keeps -inf and refers to zero: its scores are -inf, its P zero.
                const float m_old = m_run[b];
                const bool raise = __builtin_amdgcn_ballot_w64(mx > m_old + lazy_raw) != 0;
                const float m_new = raise ? max_raw(m_old, mx) : m_old;
                const float mc = m_new == -INFINITY ? 0.f : m_new * a.scale_log2e;
#pragma unroll
                for (int g = 0; g < KB32; g++) {
                    half8_t p8;
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int r = 0; r < 4; r++)
                            p8[4 * h + r] = (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[b][2 * g + h][r], a.scale_log2e, -mc));
                    pf[b][g] = p8;
                }
                if (raise) {
                    const float alpha = m_old == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_old - m_new) * a.scale_log2e);
                    m_run[b] = m_new;
#pragma unroll
                    for (int d = 0; d <= DB; d++) o[b][d] *= alpha;
                }
            }
#pragma unroll
            for (int g = 0; g < KB32; g++) {
#pragma unroll
                for (int d = 0; d < DB; d++) {
                    const half8_t vf = *reinterpret_cast<const half8_t *>(vt_lds + (16 * d + j) * VS + (((4 * g + kb) ^ swz(16 * d + j)) << 3));
#pragma unroll
                    for (int b = 0; b < QB; b++) o[b][d] = chunk_mfma16(vf, pf[b][g], o[b][d]);
                }
#pragma unroll
                for (int b = 0; b < QB; b++) o[b][DB] = chunk_mfma16(ones, pf[b][g], o[b][DB]);
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
        if (BF8 && a.causal) nf = __syncthreads_or(nf_next);
        else __syncthreads();
    }

    if (!wave_has) return;
#pragma unroll
    for (int b = 0; b < QB; b++) {
        if (qc0 + 16 * b + j >= t.cols) continue;
        const float l = o[b][DB][0];
        if constexpr (ZS) {
            const int64_t items = (int64_t)a.total_rows * a.n_q_heads, at = zr * items + item[b];
#pragma unroll
            for (int d = 0; d < DB; d++) *reinterpret_cast<float4_t *>(a.part + at * D + 16 * d + 4 * kb) = o[b][d];
            if (kb == 0) *reinterpret_cast<float2p_t *>(a.part + a.z * items * D + at * 2) = float2p_t{m_run[b], l};
        } else {
            const float inv = l == 0.f ? 0.f : 1.0f / l;          // no visible key: a zero result
#pragma unroll
            for (int d = 0; d < DB; d++) chunk_store<D, MODE>(a, item[b], 4 * d + kb, l == 0.f ? float4_t{0.f, 0.f, 0.f, 0.f} : o[b][d] * inv);
        }
    }
}

// Adds the key ranges of a column in range order; one thread per (row, head, four dims).  Rows of no sequence are
// zeroed here (fill) or left alone.
template <int D, int MODE>
__global__ __launch_bounds__(256) void chunk_merge_kernel(ChunkArgs a, int qt, int bn) {
    constexpr int DW = D / 4;
    const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t items = (int64_t)a.total_rows * a.n_q_heads;
    const int64_t item = gid / DW;
    if (item >= items) return;
    const int w4 = (int)(gid % DW), row = (int)(item / a.n_q_heads), head = (int)(item % a.n_q_heads);
    int lo = 0, hi = a.n_seq;                          // last sequence that starts at or before the row
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (chunk_clamp_row(a.cu_seqlens[mid], a.total_rows) <= row) lo = mid; else hi = mid;
    }
    const int r0 = chunk_clamp_row(a.cu_seqlens[lo], a.total_rows), r1 = max(chunk_clamp_row(a.cu_seqlens[lo + 1], a.total_rows), r0);
    if (row < r0 || row >= r1) {
        if (a.fill) chunk_store<D, MODE>(a, item, w4, float4_t{0.f, 0.f, 0.f, 0.f});
        return;
    }
    const int ctx = min(max(a.ctx_lens[lo], 0), a.max_blocks * a.block_size), p0 = ctx - (r1 - r0);
    const int cols = (r1 - r0) * a.group, col0 = ((row - r0) * a.group + head % a.group) / qt * qt;
    const int keys = a.causal ? max(p0 + (min(col0 + qt, cols) - 1) / a.group + 1, 0) : ctx;
    const int per = chunk_range_keys(keys, a.z, bn, kChunkMinKeys);
    const int used = (keys + per - 1) / per;
    const float2p_t *ml = reinterpret_cast<const float2p_t *>(a.part + a.z * items * D);
    float m = -INFINITY;
    for (int z = 0; z < used; z++) m = fmaxf(m, ml[z * items + item][0]);
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (int z = 0; z < used; z++) {
        const float2p_t x = ml[z * items + item];
        const float w = x[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x[0] - m) * a.scale_log2e);
        if (w == 0.f) continue;                        // a range of hidden keys only
        acc += *reinterpret_cast<const float4_t *>(a.part + (z * items + item) * D + 4 * w4) * w;
        l += x[1] * w;
    }
    chunk_store<D, MODE>(a, item, w4, l == 0.f ? float4_t{0.f, 0.f, 0.f, 0.f} : acc * (1.0f / l));
}

// ---- host ---------------------------------------------------------------------------------------------------------

struct ChunkShape { int qt, bn; };

static ChunkShape chunk_shape(int64_t d) {
    switch (d) {
        case 64: return {256, 64};
        case 128: return {128, 64};
        case 256: return {128, 64};
        default: return {64, 32};
    }
}

static int64_t chunk_slots(int64_t total_rows, int64_t n_seq, int64_t group, int qt) { return total_rows * group / qt + n_seq; }

// Workgroups that share a column tile: enough to give every CU two workgroups when the tiles alone do not.
static int chunk_ranges(int64_t total_rows, int64_t n_seq, int64_t n_q_heads, int64_t n_kv_heads, int64_t d, int64_t max_ctx) {
    const ChunkShape sh = chunk_shape(d);
    const int64_t tiles = chunk_slots(total_rows, n_seq, n_q_heads / n_kv_heads, sh.qt) * n_kv_heads;
    int64_t z = 512 / (tiles > 0 ? tiles : 1);
    const int64_t most = (max_ctx + kChunkMinKeys - 1) / kChunkMinKeys;
    if (z > most) z = most;
    if (z > 64) z = 64;
    return z < 1 ? 1 : (int)z;
}

template <int D, int MODE, int QB, int BN, int OCC, int WAVES, bool ALIGN4, bool ZS>
static int launch_chunk_kernel(const ChunkArgs &a, hipStream_t s) {
    constexpr int QT = 16 * QB * WAVES;
    constexpr int KS = MODE == FEATHER_E5M2 ? (D + 16) / 2 : D + 8;
    constexpr size_t lds = (size_t)(BN * KS + D * BN) * 2 * 2;
    const char *me = "feather_paged_chunk_attn_fp8";
    const int64_t slots = chunk_slots(a.total_rows, a.n_seq, a.group, QT);
    const int64_t blocks = slots * a.n_kv_heads * a.z;
    FEATHER_CHECK(blocks + kChunkFillGroups < (1ll << 31), FEATHER_ESHAPE, "%s: grid too large", me);
    auto kern = chunk_attn_kernel<D, MODE, QB, BN, OCC, WAVES, ALIGN4, ZS>;
    static unsigned long long lds_raised = 0;
    hipError_t e = raise_lds_limit(reinterpret_cast<const void *>(kern), lds, lds_raised);
    FEATHER_CHECK(e == hipSuccess, FEATHER_ELAUNCH, "%s: cannot raise LDS limit: %s", me, hipGetErrorString(e));
    hipLaunchKernelGGL(kern, dim3((unsigned)(blocks + (a.fill && !ZS ? kChunkFillGroups : 0))), dim3(64 * WAVES), lds, s, a, (int)slots, 0);
    return check_launch(me);
}

template <int D, int MODE, int QB, int BN, int OCC, int WAVES>
static int launch_chunk(const ChunkArgs &a, hipStream_t s) {
    const bool al = a.block_size % 4 == 0;
    if (a.z == 1)
        return al ? launch_chunk_kernel<D, MODE, QB, BN, OCC, WAVES, true, false>(a, s)
                  : launch_chunk_kernel<D, MODE, QB, BN, OCC, WAVES, false, false>(a, s);
    const int rc = al ? launch_chunk_kernel<D, MODE, QB, BN, OCC, WAVES, true, true>(a, s)
                      : launch_chunk_kernel<D, MODE, QB, BN, OCC, WAVES, false, true>(a, s);
    if (rc != FEATHER_OK) return rc;
    const int64_t threads = (int64_t)a.total_rows * a.n_q_heads * (D / 4);
    hipLaunchKernelGGL((chunk_merge_kernel<D, MODE>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, a, 16 * QB * WAVES, BN);
    return check_launch("feather_paged_chunk_attn_fp8 (merge of the key ranges)");
}

template <int MODE>
static int dispatch_chunk(const ChunkArgs &a, int64_t d, hipStream_t s) {
    switch (d) {
        case 64: return launch_chunk<64, MODE, 4, 64, 2, 4>(a, s);
        case 128: return launch_chunk<128, MODE, 2, 64, 2, 4>(a, s);
        case 256: return launch_chunk<256, MODE, 1, 64, 1, 8>(a, s);
        default: return launch_chunk<512, MODE, 1, 32, 1, 4>(a, s);
    }
}

}  // namespace feather

using namespace feather;

extern "C" int64_t feather_paged_chunk_attn_scratch_bytes(int64_t n_seq, int64_t total_rows, int64_t n_q_heads,
                                                          int64_t n_kv_heads, int64_t d, int64_t max_ctx,
                                                          int64_t max_q_len) {
    if (n_seq <= 0 || total_rows <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || d <= 0 || max_ctx <= 0 || max_q_len < 0) return 0;
    const int z = chunk_ranges(total_rows, n_seq, n_q_heads, n_kv_heads, d, max_ctx);
    return z > 1 ? z * total_rows * n_q_heads * (d + 2) * 4 : 0;
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
    FEATHER_CHECK(scale > 0.f && scale <= 3.0e38f, FEATHER_EINVAL,
                  "%s: scale must be positive and finite (the running maximum is kept on raw scores)", me);
    FEATHER_CHECK(block_size < (1ll << 30) && max_blocks < (1ll << 30) && max_blocks * block_size < (1ll << 30) &&
                      total_rows < (1ll << 30) && n_seq < (1ll << 30) && n_q_heads < (1ll << 20) &&
                      total_rows * n_q_heads < (1ll << 30),
                  FEATHER_ESHAPE, "%s: shape too large", me);
    FEATHER_CHECK(n_blocks * n_kv_heads < (1ll << 32) && n_blocks * n_kv_heads * block_size < (1ll << 32), FEATHER_ESHAPE,
                  "%s: the cache holds more than 2^32 rows", me);
    if (total_rows == 0) return FEATHER_OK;
    if (n_seq == 0 && !fill) return FEATHER_OK;
    FEATHER_CHECK(q && k_cache && v_cache && out && cu_seqlens && (n_seq == 0 || (ctx_lens && (block_tables || max_blocks == 0))), FEATHER_EINVAL,
                  "%s: null pointer", me);
    FEATHER_CHECK(aligned(q, 8) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(out, 16) && aligned(scratch, 16) &&
                      aligned(block_tables, 4) && aligned(cu_seqlens, 4) && aligned(ctx_lens, 4),
                  FEATHER_EINVAL, "%s: misaligned pointer", me);
    int z = n_seq > 0 ? chunk_ranges(total_rows, n_seq, n_q_heads, n_kv_heads, d, max_blocks * block_size) : 1;
    if (!scratch) z = 1;
    while (z > 1 && z * total_rows * n_q_heads * (d + 2) * 4 > scratch_bytes) z--;   // a smaller workspace: fewer ranges
    int shift = 0;
    while ((1ll << shift) < block_size) shift++;
    ChunkArgs a;
    a.q = (const uint32_t *)q; a.k_cache = (const uint32_t *)k_cache; a.v_cache = (const uint32_t *)v_cache;
    a.block_tables = (const int32_t *)block_tables; a.cu_seqlens = (const int32_t *)cu_seqlens; a.ctx_lens = (const int32_t *)ctx_lens;
    a.out = out; a.part = (float *)scratch;
    a.n_seq = (int)n_seq; a.total_rows = (int)total_rows; a.n_q_heads = (int)n_q_heads; a.n_kv_heads = (int)n_kv_heads;
    a.group = (int)(n_q_heads / n_kv_heads); a.block_size = (int)block_size; a.max_blocks = (int)max_blocks;
    a.max_blk = (uint32_t)(n_blocks - 1);
    a.div_mul = (uint32_t)((1ull << (31 + shift)) / (uint64_t)block_size + 1);
    a.div_shift = shift;
    a.causal = causal; a.z = z; a.out_kind = out_kind; a.fill = fill;
    a.scale_log2e = scale * 1.4426950408889634f;
    return mode == FEATHER_E5M2 ? dispatch_chunk<FEATHER_E5M2>(a, d, (hipStream_t)stream)
                                : dispatch_chunk<FEATHER_E4M3>(a, d, (hipStream_t)stream);
}
