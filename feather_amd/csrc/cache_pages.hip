// The pages of a paged cache as a pool on the device: ref_counts[b] counts the block-table entries (and pins of the
// caller) that hold block b, 0 = free.  Two operations, each over every cache that shares the tables (K and V of all
// layers), with no host copy of the tables and no atomics whose order shows:
//   fork     slot i of a batch goes on as a copy of slot parents[i] (beam search, samples of one prompt, reordering;
//            -1 ends the slot).  Whole blocks are shared; the block that a context ends in is copied for every child but
//            the first, because each child will write its own next token there -- and for the first too if another entry
//            or a pin holds that block, as after a length was set back into shared blocks.  Then room is reserved.
//   compact  the blocks in use move to the lowest ids, so that the upper part of the pool is free.
// Both return new tables, counts and maps and change none of those they are given.  Of the caches only blocks that no new
// row holds are written: those free before, and in a fork also those that this very call releases, so the old tables are
// void after it, also when the pool ran out.  Free blocks are handed out lowest id first in (slot, entry) order, so results
// are those of a serial loop.
//
// Integer part: every chunk of the pool is one workgroup that reads all tables once and counts in LDS, beside one
// workgroup per slot that lays out the slot's new row.  The tables and counts are read from the L2, so a read is a round
// trip: eight are in flight per thread (256 slots of 128 entries, 20480 blocks: 11 us, one at a time 17).  Chunks of 1024
// blocks, more only for a pool of more than 262144 (chunks of 4096: 11.1 us instead of 9.6, and 7.4 instead of 5.2 for
// the compaction plan of 8192 blocks: fewer workgroups, longer serial parts).
//
// Copies: 16 bytes a lane, eight caches in flight; bound by the copy rate once there is much to move.  Measured: beams of
// two requests, 512 blocks, 8 caches 4.6 + 4.9 us (plan, copies; latency only); 256 slots of which 192 go on, 44 caches
// 9.4 + 14.4 us for 23 MB (six dependent reads before the first copy); compaction of 8192 blocks, 60 % in use, 44 caches
// 5.0 + 150 us for 709 MB, 4.7 TB/s of the 5.1 that a plain copy of 1 GiB reaches.
#include "common.h"

namespace feather {

constexpr int kPgThreads = 256;
constexpr int kPgMaxCaches = 64;          // caches of one launch (their pointers travel with the kernel's arguments)
constexpr int kPgChunkThreads = 1024;
constexpr int kPgMinChunk = kPgChunkThreads, kPgMaxChunks = 256, kPgMaxChunk = 16384;
constexpr int kPgMaxSlots = 8192;

struct CachePtrs {
    u32x4 *p[kPgMaxCaches];
};

__device__ __forceinline__ int pg_block_sum(int x, int *red, int threads) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, kWave);
    __syncthreads();
    if (lane_id() == 0) red[threadIdx.x / kWave] = x;
    __syncthreads();
    int t = 0;
    for (int w = 0; w < threads / kWave; w++) t += red[w];
    return t;
}

// exclusive prefix sum over the workgroup; total in *sum
__device__ __forceinline__ int pg_block_scan(int x, int *red, int threads, int *sum) {
    int inc = x;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const int t = __shfl_up(inc, off, kWave);
        if (lane_id() >= off) inc += t;
    }
    __syncthreads();
    if (lane_id() == kWave - 1) red[threadIdx.x / kWave] = inc;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < threads / kWave; w++) {
        if (w < (int)threadIdx.x / kWave) before += red[w];
        all += red[w];
    }
    *sum = all;
    return before + inc - x;
}

// ---- fork ---------------------------------------------------------------------------------------------------------

struct ForkArgs {
    const int32_t *tables, *ctx_lens, *ref, *parents, *room;
    int32_t *tables_out, *ctx_out, *ref_out, *status;
    int32_t *need;          // [n_seq] blocks a slot asks for; bit 31: the first is the copy of its tail
    int32_t *source;        // [n_seq] block that copy is made of
    int32_t *free_count;    // [chunks] free blocks of a chunk
    int32_t *free_ids;      // [n_blocks] their ids, chunk by chunk
    int n_seq, max_blocks, block_size, n_blocks, chunk, chunks;
    uint32_t row_mul;       // i / max_blocks = umulhi(2 i, row_mul) >> row_shift for 0 <= i < 2^31
    int row_shift;
};

constexpr int kFreshTail = -2, kFreshRoom = -3;   // entries of a new row that still wait for a block

// Workgroups [0, chunks): reference counts and free blocks of a chunk of the pool.  An old row p with n children
// passes its whole blocks on to all of them, the rest of its entries to the first, but no block of the rest that is
// held by others as well (its count was above 1, a bit of `held`): an entry's count changes by n - 1, or by 0 if passed on
// and -1 if not.  Such a block under the end of a context is copied for the first child too (a bit of `source`): should its
// count come to 0, it is free only after this call.  Counts as they were decide, not those that remain when other rows have
// let go: those would be known only when all chunks are done, a third launch; the price is a copy that could be spared when
// the other holders end in the same call.  Workgroups from `chunks` on: the new row of one slot, with marks for fresh
// blocks.
__global__ __launch_bounds__(kPgChunkThreads) void fork_plan_kernel(ForkArgs a) {
    extern __shared__ __attribute__((aligned(16))) int pg_lds[];
    __shared__ int red[kPgChunkThreads / kWave];
    const int tid = threadIdx.x, cap = a.max_blocks * a.block_size;
    if ((int)blockIdx.x < a.chunks) {
        int *count = pg_lds;
        int2 *row = reinterpret_cast<int2 *>(pg_lds + a.chunk);        // children; 2 * whole blocks + (1: a part of one more)
        uint32_t *held = reinterpret_cast<uint32_t *>(row + a.n_seq), *source = held + a.chunk / 32;
        const int b0 = blockIdx.x * a.chunk, n = min(a.chunk, a.n_blocks - b0);
        for (int i = tid; i < a.chunk; i += kPgChunkThreads) {          // (a chunk is a multiple of the workgroup)
            const int r = i < n ? a.ref[b0 + i] : 0;
            const uint64_t m = __builtin_amdgcn_ballot_w64(r > 1);
            count[i] = r;
            if (lane_id() < 2) {
                held[i / 64 * 2 + lane_id()] = (uint32_t)(m >> (32 * lane_id()));
                source[i / 64 * 2 + lane_id()] = 0;
            }
        }
        for (int i = tid; i < a.n_seq; i += kPgChunkThreads) {
            const int len = min(max(a.ctx_lens[i], 0), cap);
            row[i] = int2{0, 2 * (len / a.block_size) + (len % a.block_size != 0)};
        }
        __syncthreads();
        for (int i = tid; i < a.n_seq; i += kPgChunkThreads) {
            const int p = a.parents[i];
            if ((unsigned)p < (unsigned)a.n_seq) atomicAdd(&row[p].x, 1);
        }
        __syncthreads();
        constexpr int G = 8;                           // table entries in flight per thread
        const int entries = a.n_seq * a.max_blocks;
        for (int i0 = tid; i0 < entries; i0 += G * kPgChunkThreads) {
            int v[G];
#pragma unroll
            for (int g = 0; g < G; g++) v[g] = a.tables[min(i0 + g * kPgChunkThreads, entries - 1)] - b0;
#pragma unroll
            for (int g = 0; g < G; g++) {
                const int i = i0 + g * kPgChunkThreads;
                if (i >= entries || (unsigned)v[g] >= (unsigned)n) continue;
                const int p = (int)(__umulhi(2u * (uint32_t)i, a.row_mul) >> a.row_shift), e = i - p * a.max_blocks;
                const int2 r = row[p];                 // (one read of 64 bits: the LDS bounds this loop)
                int change = r.x - 1;
                if (2 * e + 1 >= r.y) {                // not a whole block of the context
                    change = -1;
                    if (r.x > 0) {
                        const uint32_t bit = 1u << (v[g] & 31);
                        if (!(held[v[g] >> 5] & bit)) change = 0;
                        else if (2 * e + 1 == r.y) atomicOr(&source[v[g] >> 5], bit);
                    }
                }
                if (change) atomicAdd(&count[v[g]], change);
            }
        }
        __syncthreads();
        const int per = (n + kPgChunkThreads - 1) / kPgChunkThreads, i0 = min(tid * per, n), i1 = min(i0 + per, n);
        auto is_free = [&](int i) { return count[i] == 0 && !(source[i >> 5] >> (i & 31) & 1); };
        int mine = 0;
        for (int i = i0; i < i1; i++) {
            a.ref_out[b0 + i] = count[i];
            mine += is_free(i);
        }
        int total;
        int at = pg_block_scan(mine, red, kPgChunkThreads, &total);
        for (int i = i0; i < i1; i++)
            if (is_free(i)) a.free_ids[b0 + at++] = b0 + i;
        if (tid == 0) a.free_count[blockIdx.x] = total;
        return;
    }
    const int i = blockIdx.x - a.chunks, p = a.parents[i];
    const bool alive = (unsigned)p < (unsigned)a.n_seq;
    auto entry_of = [&](int e, int &v, int &count) {   // the parent's entry, -1 for what is no block, and the block's count
        v = alive && e < a.max_blocks ? a.tables[(int64_t)p * a.max_blocks + e] : -1;
        if ((unsigned)v >= (unsigned)a.n_blocks) v = -1;
        count = v >= 0 ? a.ref[v] : 0;
    };
    int v_next, count_next, earlier = 0;
    entry_of(tid, v_next, count_next);                 // requested before the vote, which waits for all earlier parents
    if (alive)
        for (int k = tid; k < i; k += kPgChunkThreads) earlier |= a.parents[k] == p;
    const int len = alive ? min(max(a.ctx_lens[p], 0), cap) : 0;
    const bool heir = !__syncthreads_or(earlier) && alive;
    const int whole = len / a.block_size, used = (len + a.block_size - 1) / a.block_size;
    const int wanted = a.room ? max(a.room[i], 0) : 0;
    const int want = wanted >= cap ? a.max_blocks : (wanted + a.block_size - 1) / a.block_size;
    int fresh = 0, hole = 0, tail = 0;
    for (int e = tid; e < a.max_blocks; e += kPgChunkThreads) {
        int v = v_next;
        const bool own = heir && (e < whole || count_next <= 1);   // may stay in the slot's row as it is
        entry_of(e + kPgChunkThreads, v_next, count_next);
        if (e < used) {
            hole |= v < 0;
            if (!own && e == whole && v >= 0) {
                a.source[i] = v;
                v = kFreshTail;
                tail = 1;
            }
        } else {
            if (!own) v = -1;
            if (v < 0 && e < want) v = kFreshRoom;
        }
        fresh += v < -1;
        a.tables_out[(int64_t)i * a.max_blocks + e] = v;
    }
    hole = __syncthreads_or(hole);
    tail = __syncthreads_or(tail);
    const int sum = pg_block_sum(fresh, red, kPgChunkThreads);
    if (tid == 0) {
        a.need[i] = sum | (tail ? (int)0x80000000 : 0);
        a.ctx_out[i] = len;
        if (a.status) a.status[i] = hole ? 2 : (wanted > cap ? 1 : 0);
    }
}

// rank of slot i's first fresh block, the chunk prefix in LDS, and the id of the k-th free block
struct FreeLookup {
    int *before;            // [chunks + 1] free blocks in front of a chunk
    const ForkArgs *a;
    __device__ int id(int k) const {
        if (k >= before[a->chunks]) return -1;
        int lo = 0, hi = a->chunks;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (before[mid] <= k) lo = mid; else hi = mid;
        }
        return a->free_ids[lo * a->chunk + k - before[lo]];
    }
};

// Workgroups (i, 0): the fresh blocks of slot i.  Workgroups (i, 1 + g): the copy of its tail in eight caches.
__global__ __launch_bounds__(kPgThreads) void fork_assign_kernel(ForkArgs a, CachePtrs caches, int n_caches, int units, int assign) {
    __shared__ int red[kPgThreads / kWave];
    __shared__ int before[kPgMaxChunks + 1];
    const int tid = threadIdx.x, i = blockIdx.x;
    const int need = a.need[i], tail = need < 0, count = need & 0x7FFFFFFF;
    const bool copies = !assign || blockIdx.y > 0;
    if (copies ? !tail : count == 0) return;
    int part = 0;
    for (int k = tid; k < i; k += kPgThreads) part += a.need[k] & 0x7FFFFFFF;
    const int first = pg_block_sum(part, red, kPgThreads);
    int sum;
    const int mine = tid < a.chunks ? a.free_count[tid] : 0;
    const int ex = pg_block_scan(mine, red, kPgThreads, &sum);
    if (tid < a.chunks) before[tid] = ex;
    if (tid == 0) before[a.chunks] = sum;
    __syncthreads();
    const FreeLookup look = {before, &a};
    if (!copies) {
        int32_t *row = a.tables_out + (int64_t)i * a.max_blocks;
        int done = 0, short_of = 0;
        for (int e0 = 0; e0 < a.max_blocks; e0 += kPgThreads) {
            const int e = e0 + tid, v = e < a.max_blocks ? row[e] : -1;
            int all;
            const int rank = pg_block_scan(v < -1 ? 1 : 0, red, kPgThreads, &all);
            if (v < -1) {
                const int id = look.id(first + done + rank);
                row[e] = id;
                if (id >= 0) a.ref_out[id] = 1;
                else {
                    short_of = 1;
                    if (v == kFreshTail) a.ctx_out[i] = a.ctx_out[i] / a.block_size * a.block_size;   // holds its whole blocks only
                }
            }
            done += all;
        }
        short_of = __syncthreads_or(short_of);
        if (tid == 0 && short_of && a.status) a.status[i] = 3;
        return;
    }
    const int to = look.id(first);                    // the tail is the first fresh entry of a row
    if (to < 0) return;
    const int64_t src = (int64_t)a.source[i] * units, dst = (int64_t)to * units;
    const int c0 = (blockIdx.y - (assign ? 1 : 0)) * 8;
    for (int u = tid; u < units; u += kPgThreads) {
        u32x4 x[8];
#pragma unroll
        for (int c = 0; c < 8; c++) x[c] = caches.p[min(c0 + c, n_caches - 1)][src + u];
#pragma unroll
        for (int c = 0; c < 8; c++)
            if (c0 + c < n_caches) caches.p[c0 + c][dst + u] = x[c];
    }
}

// ---- compact ------------------------------------------------------------------------------------------------------

struct CompactArgs {
    const int32_t *tables, *ref;
    int32_t *tables_out, *ref_out, *block_map, *n_live;
    int32_t *rank;          // [n_blocks] of a hole (free, below n_live): holes before it; of a high block (used, not below n_live): used blocks after it
    int32_t *holes, *highs; // [n_blocks] by rank
    int32_t *moves;         // [1]
    int64_t entries;
    int n_blocks, chunk;
};

// One workgroup per chunk.  Each counts the used blocks before its chunk and in the whole pool by itself (the counts
// of a pool fit the L2), so no second pass over partial sums is needed.  The r-th hole from below takes the r-th high
// block from above.
__global__ __launch_bounds__(kPgChunkThreads) void compact_plan_kernel(CompactArgs a) {
    __shared__ int red[kPgChunkThreads / kWave];
    const int tid = threadIdx.x, b0 = blockIdx.x * a.chunk, n = min(a.chunk, a.n_blocks - b0);
    int before = 0, all = 0;
    constexpr int G = 8;                               // counts in flight per thread
    for (int i0 = tid; i0 < a.n_blocks; i0 += G * kPgChunkThreads) {
        int v[G];
#pragma unroll
        for (int g = 0; g < G; g++) v[g] = a.ref[min(i0 + g * kPgChunkThreads, a.n_blocks - 1)];
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int i = i0 + g * kPgChunkThreads, used = i < a.n_blocks && v[g] > 0;
            all += used;
            before += i < b0 ? used : 0;
        }
    }
    before = pg_block_sum(before, red, kPgChunkThreads);
    all = pg_block_sum(all, red, kPgChunkThreads);
    const int per = (n + kPgChunkThreads - 1) / kPgChunkThreads, i0 = min(tid * per, n), i1 = min(i0 + per, n);
    int mine = 0;
    for (int i = i0; i < i1; i++) mine += a.ref[b0 + i] > 0;
    int sum;
    int used_before = before + pg_block_scan(mine, red, kPgChunkThreads, &sum);
    for (int i = i0; i < i1; i++) {
        const int b = b0 + i, used = a.ref[b] > 0;
        if (b == all) *a.moves = all - used_before;   // used blocks from n_live on
        if (!used && b < all) {
            const int r = b - used_before;
            a.rank[b] = r;
            a.holes[r] = b;
        }
        if (used && b >= all) {
            const int r = all - 1 - used_before;
            a.rank[b] = r;
            a.highs[r] = b;
        }
        used_before += used;
    }
    if (blockIdx.x == 0 && tid == 0) {
        *a.n_live = all;
        if (all == a.n_blocks) *a.moves = 0;
    }
}

__global__ __launch_bounds__(kPgThreads) void compact_move_kernel(CompactArgs a, CachePtrs caches, int n_caches, int units, int index_groups) {
    const int moves = *a.moves;
    if ((int)blockIdx.x < index_groups) {
        const int live = *a.n_live, step = index_groups * kPgThreads, first = blockIdx.x * kPgThreads + threadIdx.x;
        auto moved = [&](int b) { return b < live ? b : a.holes[a.rank[b]]; };
        for (int b = first; b < a.n_blocks; b += step) {
            const int r = a.ref[b];
            a.block_map[b] = r > 0 ? moved(b) : -1;
            a.ref_out[b] = b >= live ? 0 : (r > 0 ? r : a.ref[a.highs[a.rank[b]]]);
        }
        for (int64_t i = first; i < a.entries; i += step) {
            const int v = a.tables[i];
            a.tables_out[i] = (unsigned)v < (unsigned)a.n_blocks && a.ref[v] > 0 ? moved(v) : -1;
        }
        return;
    }
    // a workgroup's share of the (move, eight caches) items
    const int groups = (n_caches + 7) / 8;
    for (int64_t it = blockIdx.x - index_groups; it < (int64_t)moves * groups; it += gridDim.x - index_groups) {
        const int m = (int)(it / groups), c0 = (int)(it - (int64_t)m * groups) * 8;
        const int64_t src = (int64_t)a.highs[m] * units, dst = (int64_t)a.holes[m] * units;
        for (int u = threadIdx.x; u < units; u += kPgThreads) {
            u32x4 x[8];
#pragma unroll
            for (int c = 0; c < 8; c++) x[c] = caches.p[min(c0 + c, n_caches - 1)][src + u];
#pragma unroll
            for (int c = 0; c < 8; c++)
                if (c0 + c < n_caches) caches.p[c0 + c][dst + u] = x[c];
        }
    }
}

static int64_t pg_chunk(int64_t n_blocks) {
    int64_t c = kPgMinChunk;
    while (c < kPgMaxChunk && (n_blocks + c - 1) / c > kPgMaxChunks) c *= 2;
    return c;
}

static int pg_check_caches(const char *me, const void *const *caches, int64_t n_caches, int64_t block_bytes, int64_t n_blocks) {
    FEATHER_CHECK(n_caches >= 0 && n_caches <= (1 << 20) && (caches || n_caches == 0), FEATHER_EINVAL, "%s: bad list of caches", me);
    FEATHER_CHECK(block_bytes > 0 && block_bytes % 16 == 0 && block_bytes < (1ll << 33), FEATHER_ESHAPE,
                  "%s: a block of %lld bytes is not a multiple of 16", me, (long long)block_bytes);
    FEATHER_CHECK(n_blocks >= 1 && (n_blocks + kPgMaxChunk - 1) / kPgMaxChunk <= kPgMaxChunks, FEATHER_ESHAPE,
                  "%s: n_blocks=%lld outside [1, %d]", me, (long long)n_blocks, kPgMaxChunk * kPgMaxChunks);
    for (int64_t c = 0; c < n_caches; c++)
        FEATHER_CHECK(caches[c] && aligned(caches[c], 16), FEATHER_EINVAL, "%s: cache %lld is null or misaligned", me, (long long)c);
    return FEATHER_OK;
}

static CachePtrs pg_ptrs(const void *const *caches, int64_t first, int64_t n) {
    CachePtrs p;
    for (int i = 0; i < kPgMaxCaches; i++) p.p[i] = i < n ? (u32x4 *)const_cast<void *>(caches[first + i]) : nullptr;
    return p;
}

}  // namespace feather

using namespace feather;

extern "C" int64_t feather_paged_cache_fork_scratch_bytes(int64_t n_seq, int64_t n_blocks) {
    if (n_seq < 0 || n_blocks < 0) return 0;
    return (2 * n_seq + kPgMaxChunks + n_blocks) * 4;
}

extern "C" int feather_paged_cache_fork(const void *const *caches_host, int64_t n_caches, int64_t block_bytes,
                                        const void *block_tables, const void *ctx_lens, const void *ref_counts,
                                        const void *parents, const void *room, void *tables_out, void *ctx_out, void *ref_out,
                                        void *seq_status, void *scratch, int64_t n_seq, int64_t max_blocks, int64_t block_size,
                                        int64_t n_blocks, void *stream) {
    const char *me = "feather_paged_cache_fork";
    int rc = pg_check_caches(me, caches_host, n_caches, block_bytes, n_blocks);
    if (rc != FEATHER_OK) return rc;
    FEATHER_CHECK(n_seq >= 0 && max_blocks >= 0 && block_size > 0, FEATHER_EINVAL, "%s: bad shape", me);
    FEATHER_CHECK(n_seq <= kPgMaxSlots, FEATHER_ESHAPE, "%s: n_seq=%lld above %d", me, (long long)n_seq, kPgMaxSlots);
    FEATHER_CHECK(max_blocks < (1ll << 30) && block_size < (1ll << 30) && max_blocks * block_size < (1ll << 30) &&
                      n_seq * max_blocks < (1ll << 30),
                  FEATHER_ESHAPE, "%s: shape too large", me);
    FEATHER_CHECK(ref_counts && ref_out && scratch && ref_counts != ref_out, FEATHER_EINVAL, "%s: null pointer, or ref_out is ref_counts", me);
    FEATHER_CHECK(n_seq == 0 || (ctx_lens && parents && ctx_out && ctx_out != ctx_lens), FEATHER_EINVAL,
                  "%s: null pointer, or ctx_out is ctx_lens", me);
    FEATHER_CHECK(n_seq * max_blocks == 0 || (block_tables && tables_out && tables_out != block_tables), FEATHER_EINVAL,
                  "%s: null pointer, or tables_out is block_tables", me);
    FEATHER_CHECK(aligned(block_tables, 4) && aligned(ctx_lens, 4) && aligned(ref_counts, 4) && aligned(parents, 4) && aligned(room, 4) &&
                      aligned(tables_out, 4) && aligned(ctx_out, 4) && aligned(ref_out, 4) && aligned(seq_status, 4) && aligned(scratch, 4),
                  FEATHER_EINVAL, "%s: misaligned pointer", me);
    ForkArgs a;
    a.tables = (const int32_t *)block_tables; a.ctx_lens = (const int32_t *)ctx_lens; a.ref = (const int32_t *)ref_counts;
    a.parents = (const int32_t *)parents; a.room = (const int32_t *)room; a.tables_out = (int32_t *)tables_out;
    a.ctx_out = (int32_t *)ctx_out; a.ref_out = (int32_t *)ref_out; a.status = (int32_t *)seq_status;
    a.need = (int32_t *)scratch; a.source = a.need + n_seq; a.free_count = a.source + n_seq; a.free_ids = a.free_count + kPgMaxChunks;
    a.n_seq = (int)n_seq; a.max_blocks = (int)max_blocks; a.block_size = (int)block_size; a.n_blocks = (int)n_blocks;
    a.chunk = (int)pg_chunk(n_blocks); a.chunks = (int)((n_blocks + a.chunk - 1) / a.chunk);
    const size_t lds = ((size_t)a.chunk + 2 * n_seq + a.chunk / 16) * 4;   // counts, two words per slot, two bits per block
    a.row_shift = 0;
    while ((1ll << a.row_shift) < max_blocks) a.row_shift++;
    a.row_mul = max_blocks > 0 ? (uint32_t)((1ull << (31 + a.row_shift)) / (uint64_t)max_blocks + 1) : 0;
    static unsigned long long lds_raised = 0;
    hipError_t e = raise_lds_limit(reinterpret_cast<const void *>(fork_plan_kernel), (size_t)(kPgMaxChunk + 2 * kPgMaxSlots + kPgMaxChunk / 16) * 4, lds_raised);
    FEATHER_CHECK(e == hipSuccess, FEATHER_ELAUNCH, "%s: cannot raise LDS limit: %s", me, hipGetErrorString(e));
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(fork_plan_kernel, dim3((unsigned)(a.chunks + n_seq)), dim3(kPgChunkThreads), lds, s, a);
    rc = check_launch(me);
    if (rc != FEATHER_OK || n_seq == 0) return rc;
    for (int64_t c0 = 0; c0 == 0 || c0 < n_caches; c0 += kPgMaxCaches) {   // the first launch also hands out the blocks
        const int64_t n = n_caches - c0 < kPgMaxCaches ? n_caches - c0 : kPgMaxCaches;
        const int assign = c0 == 0;
        hipLaunchKernelGGL(fork_assign_kernel, dim3((unsigned)n_seq, (unsigned)((n + 7) / 8 + assign)), dim3(kPgThreads), 0, s, a,
                           pg_ptrs(caches_host, c0, n), (int)n, (int)(block_bytes / 16), assign);
        rc = check_launch(me);
        if (rc != FEATHER_OK) return rc;
    }
    return FEATHER_OK;
}

extern "C" int64_t feather_paged_cache_compact_scratch_bytes(int64_t n_blocks) { return n_blocks < 0 ? 0 : (3 * n_blocks + 1) * 4; }

extern "C" int feather_paged_cache_compact(const void *const *caches_host, int64_t n_caches, int64_t block_bytes,
                                           const void *block_tables, const void *ref_counts, void *tables_out, void *ref_out,
                                           void *block_map, void *n_live, void *scratch, int64_t n_entries, int64_t n_blocks,
                                           void *stream) {
    const char *me = "feather_paged_cache_compact";
    int rc = pg_check_caches(me, caches_host, n_caches, block_bytes, n_blocks);
    if (rc != FEATHER_OK) return rc;
    FEATHER_CHECK(n_entries >= 0 && n_entries < (1ll << 40), FEATHER_EINVAL, "%s: bad shape", me);
    FEATHER_CHECK(ref_counts && ref_out && block_map && n_live && scratch && ref_counts != ref_out, FEATHER_EINVAL,
                  "%s: null pointer, or ref_out is ref_counts", me);
    FEATHER_CHECK(n_entries == 0 || (block_tables && tables_out), FEATHER_EINVAL, "%s: null pointer", me);
    FEATHER_CHECK(aligned(block_tables, 4) && aligned(ref_counts, 4) && aligned(tables_out, 4) && aligned(ref_out, 4) &&
                      aligned(block_map, 4) && aligned(n_live, 4) && aligned(scratch, 4),
                  FEATHER_EINVAL, "%s: misaligned pointer", me);
    CompactArgs a;
    a.tables = (const int32_t *)block_tables; a.ref = (const int32_t *)ref_counts; a.tables_out = (int32_t *)tables_out;
    a.ref_out = (int32_t *)ref_out; a.block_map = (int32_t *)block_map; a.n_live = (int32_t *)n_live;
    a.moves = (int32_t *)scratch; a.rank = a.moves + 1; a.holes = a.rank + n_blocks; a.highs = a.holes + n_blocks;
    a.entries = n_entries; a.n_blocks = (int)n_blocks; a.chunk = (int)pg_chunk(n_blocks);
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(compact_plan_kernel, dim3((unsigned)((n_blocks + a.chunk - 1) / a.chunk)), dim3(kPgChunkThreads), 0, s, a);
    rc = check_launch(me);
    if (rc != FEATHER_OK) return rc;
    const int64_t most = (n_blocks > n_entries ? n_blocks : n_entries);
    const int64_t index = (most + kPgThreads - 1) / kPgThreads;
    for (int64_t c0 = 0; c0 == 0 || c0 < n_caches; c0 += kPgMaxCaches) {
        const int64_t n = n_caches - c0 < kPgMaxCaches ? n_caches - c0 : kPgMaxCaches;
        const int groups = c0 == 0 ? (int)(index < 1024 ? index : 1024) : 0;
        const int64_t items = n_blocks / 2 * ((n + 7) / 8);               // at most half of the pool moves
        const int64_t copies = items < 2048 ? items : 2048;
        if (groups + copies == 0) continue;
        hipLaunchKernelGGL(compact_move_kernel, dim3((unsigned)(groups + copies)), dim3(kPgThreads), 0, s, a, pg_ptrs(caches_host, c0, n),
                           (int)n, (int)(block_bytes / 16), groups);
        rc = check_launch(me);
        if (rc != FEATHER_OK) return rc;
    }
    return FEATHER_OK;
}
