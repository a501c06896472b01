// Decode attention of many sequences over one paged pool: one query row per sequence and head, each sequence behind its
// own row of page ids and of its own length, the lengths on the device.
//
//   out[i, h] = sum_t p_t V[t] / sum_t p_t,  p_t = exp(q[i, h] . K[t] / sqrt(hd)),  t < lens[i]
//
// Bound by the bytes of the cache, which are read once: 4 hd lens[i] a KV head (FP16) for 4 hd lens[i] flops a query
// head. So what counts is that the memory system has enough requests from the first microsecond to the last, whatever
// the lengths are:
//   deal     The work is the list of units (sequence, KV head, page) in that order, cut into 512 runs of equal
//            length, one for each workgroup ("worker"): two workgroups of four waves for each compute unit, all resident
//            at once. Nothing is sized by the longest sequence and nothing depends on the host knowing a length. Each
//            worker finds its run by a prefix sum over the lengths (4 bytes a sequence), looks its page ids up into LDS
//            256 at a time, and then only reads pages. A unit is 16 KB of K and 16 KB of V at 128 channels: fewer
//            positions would cut rows into more partial states than they save in balance. More workers, 768 or 1024,
//            with or without more of them resident, or a last quarter of the work dealt to 512 smaller ones, are no
//            faster on long caches (146 to 154 us against 146 at 32 x 13400 positions) and up to 45 % slower
//            on short ones, through their partial states.
//   stream   Of a page each wave takes sixteen positions. Its loads are buffer loads bounded by the positions in use:
//            what lies past them (or behind a bad page id) is not read and comes as zeros, and since every item, an
//            empty one behind the last too, issues the same loads, the compiler can count them: the next two items'
//            loads are in flight while one is computed (one: the same to 3 % slower; three: 10 to 25 % slower).
//            They are non-temporal (a plain read of 512 MB runs at 6.7 TB/s so, at 5.9 without).
//   products S = K Q^T (16x16x32, sixteen positions by up to sixteen query heads of the group), the softmax online per
//            head in FP32, O^T = V^T P^T (16x16x16). V's share of the operand is picked from the registers; K takes a
//            turn through the wave's own LDS (struct Block).
//   join     Where a run ends a row (sequence, KV head) the four waves' states meet in LDS. A row that lies
//            wholly inside a worker is finished there; otherwise each worker leaves (sum of p V, maximum, sum of p) in
//            `parts`, and a second launch folds them in the order of their pages.
// Measured at 28 + 4 heads of 128 (both launches, from events around passes over three caches in turn): 1 x 14449
// positions 14.7 us, 8 x 2048 13.8, 24 of 0 .. 14449 65 us (5.5 TB/s), 32 of 12345 .. 14449 147.3 us (5.9 TB/s, 93 % of
// what a plain read of 256-byte vectors reaches; the first launch alone 144 us, 6.1); 64 of 6001 .. 8192 in E4M3 85.4 us
// (5.5 TB/s). What is left below 100 MB is latency: 3.2 us until a worker's first loads go out (its arguments, the lengths -
// of which a thread asks for four one after another, each awaited, from four sequences on -, the page ids), 3 until they
// are back, and 4.4 for the second launch.
#include <algorithm>

#include "attn_common.hpp"

namespace vv {
namespace {

constexpr int kBatchThreads = 256;
constexpr int kBatchWaves = kBatchThreads / kWave;
constexpr int kWorkers = 512;
constexpr int kSliceHeads = 16;              // query heads of a group that one workgroup takes: a matrix tile's columns
constexpr int kSeqChunk = 1024;              // sequences whose lengths a workgroup holds at a time
// A probability is rounded to FP16 for the matrix product (half a step, 2^-11 of it; the row's sum takes it unrounded).
// It is formed on the scale 2^kLift of the row's maximum, so that it leaves FP16's normal range only 2^24 below that;
// the factor is in the row's sum too and cancels.
constexpr float kLift = 10.0f;
constexpr int kDepth = 2;                    // items whose loads are in flight while one is computed
constexpr int kItems = 256;                  // pages whose work a workgroup holds at a time

struct Row {                                 // a row of the work: (sequence, KV head)
    int first, last;                         // the workers it is dealt to
};
struct BatchArgs {
    const h16* q;
    const void* k;
    const void* v;
    const int* tables;
    const int* lens;
    h16* out;
    Row* rows;              // [n_seqs * n_kv_heads]
    float* parts;
    int n_q_heads, n_kv_heads, n_seqs, max_pages, n_pages;
    float scale_log2;
};

// A score's product with the softmax's scale, rounded by itself. Fused into the subtraction of the maximum (which was
// rounded), the largest score's exponent would be off by half a step of the score: 8 at 2^27, which FP16 inputs reach
// (65504^2 sqrt(128) log2(e) is 2^36), and the probability past what FP16 holds. Rounded first, the largest score is its
// maximum to the bit.
__device__ __forceinline__ float scaled(float score, float scale) {
#pragma clang fp contract(off)
    return score * scale;
}

__device__ __forceinline__ int seen_len(const BatchArgs& a, int s) { return min(max(a.lens[s], 0), a.max_pages * kPage); }
__device__ __forceinline__ int pages_of(int len) { return (len + kPage - 1) / kPage; }

template <int kCtrl, int kRows>
__device__ __forceinline__ int add_lane(int v) { return v + __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xF, false); }
// Inclusive prefix over the wave, in the vector ALU: shifts by 1, 2, 4, 8 within rows of sixteen lanes, then the last
// lane of a row into the next row, then of the first half into the second.
__device__ __forceinline__ int wave_prefix(int v) {
    v = add_lane<0x111, 0xF>(v);
    v = add_lane<0x112, 0xF>(v);
    v = add_lane<0x114, 0xF>(v);
    v = add_lane<0x118, 0xF>(v);
    v = add_lane<0x142, 0xA>(v);
    return add_lane<0x143, 0xC>(v);
}
// Exclusive prefix over the workgroup and the sum of all. `sums` is free again after the caller's next barrier.
__device__ __forceinline__ int block_prefix(int v, int* sums, int& total) {
    const int incl = wave_prefix(v);
    if (lane_id() == 63) sums[wave_in_block()] = incl;
    __syncthreads();
    int before = incl - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < kBatchWaves; ++w) {
        if (w < wave_in_block()) before += sums[w];
        total += sums[w];
    }
    return before;
}

// The units (sequence, KV head, page), in that order, dealt to kWorkers workgroups: contiguous runs, the first
// units % kWorkers of them one longer.
struct Deal {
    int q, r;
    __device__ __forceinline__ explicit Deal(int units) : q(units / kWorkers), r(units % kWorkers) {}
    __device__ __forceinline__ int begin(int worker) const { return worker * q + min(worker, r); }
    __device__ __forceinline__ int worker_of(int unit) const {
        const int longer = r * (q + 1);
        return unit < longer ? unit / (q + 1) : r + (unit - longer) / max(q, 1);
    }
};

// Eight FP8 codes as the FP16 values they are, by the hardware's own conversion (a bit-by-bit widening of the 64 codes
// a lane holds of sixteen positions was two thirds of the loop's vector instructions and bounded it).
template <int kFmt>
__device__ __forceinline__ h16x8 widen8(uint32_t a, uint32_t b) {
    h16x8 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = i < 2 ? a : b;
        h16x2 v;
        if constexpr (kFmt == kFmtE4M3) v = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                                                  : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        else v = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, true)
                       : __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, 1.0f, false);
        out[2 * i] = v[0];
        out[2 * i + 1] = v[1];
    }
    return out;
}

// One page of a worker's run, ready to be fetched.
struct __attribute__((aligned(16))) Item {
    int page;        // a page of the pool; 0 where the table names none
    int meta;        // positions in use (0 .. 64), then the flags
    int seq, kvh;
};
constexpr int kFirst = 1 << 8;        // begins a stretch of one row
constexpr int kLast = 1 << 9;         // ends it
constexpr int kBegun = 1 << 10;       // the row begins in this worker
constexpr int kEnded = 1 << 11;       // and ends in it

constexpr int part_floats(int hd) { return hd + 4; }       // a head's partial state: channels, max, sum, 2 unused

// A wave's sixteen positions of a page, as loaded: every load covers whole vectors, 16 bytes a lane. A vector of 256
// bytes takes sixteen lanes: load i brings positions 4 j + i, j = lane / 16. One of 128 bytes takes eight: load i
// brings positions 8 i + lane / 8. (Loads in the matrix operand's own layout, sixteen vectors by 64 bytes, stream the
// cache at 5.0 TB/s - 5.6 without the non-temporal hint - where these reach 6.4.)
template <int kHd, int kFmt>
struct Block {
    static constexpr int kUnit = kFmt == kFmtFp16 ? 2 : 1;
    static constexpr int kRow = kHd * kUnit;              // bytes per vector: 128 or 256
    static constexpr int kLoads = kRow / 64;
    static constexpr int kRowChunks = kRow / 16;
    Chunk k[kLoads], v[kLoads];
};

// A bounded view of memory for buffer loads: a lane whose offset reaches `bytes` or beyond gets zeros and touches nothing.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t bounded(const void* p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
constexpr int kNonTemporal = 2;          // the cache is read once
__device__ __forceinline__ Chunk load16(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    return __builtin_bit_cast(Chunk, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, kNonTemporal));
}

template <int kHd, int kFmt>
__global__ __launch_bounds__(kBatchThreads, 2) void decode_batch(BatchArgs a) {
    typedef Block<kHd, kFmt> B;
    constexpr int kSteps = kHd / 32;                       // 32-channel steps of the score product
    constexpr bool kNarrow = B::kRow == 128;
    constexpr int kTiles = kHd / 16;                       // O^T tiles
    constexpr int kStride = kHd + 4;
    __shared__ __attribute__((aligned(16))) float o_lds[kBatchWaves][kSliceHeads * kStride];
    __shared__ float m_lds[kBatchWaves][16], l_lds[kBatchWaves][16];
    __shared__ Chunk k_lds[kBatchWaves][16 * B::kRowChunks];
    __shared__ int s_before[kSeqChunk + 1], s_len[kSeqChunk], s_sum[kBatchWaves], s_sum2[kBatchWaves];
    __shared__ Item s_item[kItems + 2 * kDepth];

    const int tid = (int)threadIdx.x, lane = tid & 63, wave = wave_in_block();
    const int c = lane & 15, j = lane >> 4;
    const int worker = (int)blockIdx.x, slice = (int)blockIdx.y;
    const int group = a.n_q_heads / a.n_kv_heads;
    const int heads = min(kSliceHeads, group - slice * kSliceHeads);      // of this slice
    const uint32_t row_bytes = (uint32_t)a.n_kv_heads * B::kRow;

    // More sequences than are held at a time: their pages are summed beforehand.
    int total = 0;
    if (a.n_seqs > kSeqChunk) {
        int mine = 0;
        for (int s = tid; s < a.n_seqs; s += kBatchThreads) mine += pages_of(seen_len(a, s));
        block_prefix(mine, s_sum2, total);
    }

    // The lane's place inside a page, from the vector of the first row and this KV head, for load 0; load i is kLoadRows
    // rows further.
    constexpr int kLoadRows = kNarrow ? 8 : 1;
    const int chunk = lane % B::kRowChunks, row_at = kNarrow ? lane / 8 : 4 * j;
    uint32_t off[B::kLoads];
#pragma unroll
    for (int i = 0; i < B::kLoads; ++i) off[i] = (uint32_t)(16 * wave + row_at + i * kLoadRows) * row_bytes + 16u * chunk;
    // K goes through the wave's own LDS into the matrix operand's layout. Chunk x of position n sits in slot
    // x ^ n of its row (128-byte rows: x ^ n / 2), so that sixteen lanes write, and read, sixteen different slots.
    auto k_slot = [&](int n, int x) {
        return n * B::kRowChunks + (kNarrow ? x ^ ((n >> 1) & 7) : x ^ n);
    };
    // The position behind index n of the products: where two loads bring a lane's four positions they are 2 j, 2 j + 1,
    // 8 + 2 j and 9 + 2 j.
    auto position = [&](int n) { return kNarrow ? 8 * ((n >> 1) & 1) + 2 * (n >> 2) + (n & 1) : n; };

    B buf[kDepth];
    h16x8 qn[kDepth][kSteps], qf[kSteps];
    f32x4 o[kTiles];
    float m = -INFINITY, l = 0.0f;

    int chunk_units0 = 0;                                  // units before this chunk of sequences
    for (int c0 = 0; c0 < a.n_seqs; c0 += kSeqChunk) {
        constexpr int kPer = kSeqChunk / kBatchThreads;
        int len[kPer], mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int s = c0 + tid * kPer + i;
            len[i] = s < a.n_seqs ? seen_len(a, s) : 0;
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) mine += pages_of(len[i]);
        int chunk_pages;
        int before = block_prefix(mine, s_sum, chunk_pages);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            s_before[tid * kPer + i] = before;
            s_len[tid * kPer + i] = len[i];
            before += pages_of(len[i]);
        }
        if (tid == 0) s_before[kSeqChunk] = chunk_pages;
        if (a.n_seqs <= kSeqChunk) total = chunk_pages;
        const Deal deal(total * a.n_kv_heads);
        const int u0 = deal.begin(worker), u1 = deal.begin(worker + 1);
        __syncthreads();

        // Sequences without positions: zeros, and a row that nobody shares.
        for (int s = worker; s < kSeqChunk && c0 + s < a.n_seqs; s += kWorkers) {
            if (s_len[s] > 0) continue;
            for (int i = tid; i < heads * a.n_kv_heads * kHd; i += kBatchThreads) {
                const int kvh = i / (heads * kHd), e = i - kvh * heads * kHd;
                a.out[((size_t)(c0 + s) * a.n_q_heads + kvh * group + slice * kSliceHeads) * kHd + e] = (h16)0.0f;
            }
            if (slice == 0)
                for (int i = tid; i < a.n_kv_heads; i += kBatchThreads)
                    a.rows[(size_t)(c0 + s) * a.n_kv_heads + i] = Row{0, 0};
        }

        const int chunk_units1 = chunk_units0 + chunk_pages * a.n_kv_heads;
        const int last_unit = min(u1, chunk_units1);
        for (int base = max(u0, chunk_units0); base < last_unit; base += kItems) {
            const int n = min(kItems, last_unit - base);
            if (tid < 2 * kDepth) s_item[n + tid] = Item{0, 0, 0, 0};      // nothing to fetch, nothing to do
            if (tid < n) {
                const int u = base + tid, in_chunk = u - chunk_units0;
                int lo = 0, hi = min(kSeqChunk, a.n_seqs - c0) - 1;      // the first sequence that ends past the unit
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (s_before[mid + 1] * a.n_kv_heads > in_chunk) hi = mid;
                    else lo = mid + 1;
                }
                const int n_row = s_before[lo + 1] - s_before[lo];
                const int rel = in_chunk - s_before[lo] * a.n_kv_heads;
                const int kvh = rel / n_row, p = rel - kvh * n_row;
                const int row0 = u - p;                    // the row's first unit
                int page = a.tables[(size_t)(c0 + lo) * a.max_pages + p];
                int meta = min(kPage, s_len[lo] - p * kPage);
                if (page < 0 || page >= a.n_pages) page = meta = 0;
                if (p == 0 || u == u0) meta |= kFirst;
                if (p == n_row - 1 || u == u1 - 1) meta |= kLast;
                if (row0 >= u0) meta |= kBegun;
                if (row0 + n_row <= u1) meta |= kEnded;
                s_item[tid] = Item{page, meta, c0 + lo, kvh};
                if (p == 0 && slice == 0)
                    a.rows[(size_t)(c0 + lo) * a.n_kv_heads + kvh] = Row{worker, deal.worker_of(row0 + n_row - 1)};
            }
            __syncthreads();

            auto item_at = [&](int i) {
                const Item it = s_item[i];
                Item u;
                u.page = __builtin_amdgcn_readfirstlane(it.page);
                u.meta = __builtin_amdgcn_readfirstlane(it.meta);
                u.seq = __builtin_amdgcn_readfirstlane(it.seq);
                u.kvh = __builtin_amdgcn_readfirstlane(it.kvh);
                return u;
            };
            // The positions in use bound the view: what lies past them reads as zeros, and an item of none reads nothing,
            // so every item, an empty one behind the last too, issues the same loads and the waits can be counted.
            auto fetch = [&](B& b, h16x8 (&q)[kSteps], int i) {
                const Item it = item_at(i);
                const size_t at = (size_t)it.page * kPage * row_bytes + (size_t)it.kvh * B::kRow;
                const int bytes = max((it.meta & 0xFF) * (int)row_bytes - it.kvh * B::kRow, 0);
                const auto kp = bounded(static_cast<const char*>(a.k) + at, bytes);
                const auto vp = bounded(static_cast<const char*>(a.v) + at, bytes);
#pragma unroll
                for (int x = 0; x < B::kLoads; ++x) b.k[x] = load16(kp, off[x]);
#pragma unroll
                for (int x = 0; x < B::kLoads; ++x) b.v[x] = load16(vp, off[x]);
                if (it.meta & kFirst) {
                    const int head = it.kvh * group + slice * kSliceHeads + min(c, heads - 1);
                    const Chunk* qp = reinterpret_cast<const Chunk*>(a.q + ((size_t)it.seq * a.n_q_heads + head) * kHd);
#pragma unroll
                    for (int s = 0; s < kSteps; ++s)
                        q[s] = __builtin_bit_cast(h16x8, load_chunk(qp + (kFmt == kFmtFp16 ? 4 * s + j : 4 * j + s)));
                }
            };
            auto step = [&](const B& b, const h16x8 (&q)[kSteps], int i) {
                const Item it = item_at(i);
                const int in_use = (it.meta & 0xFF) - 16 * wave;       // of this wave's sixteen
                if (it.meta & kFirst) {
#pragma unroll
                    for (int s = 0; s < kSteps; ++s) qf[s] = q[s];
#pragma unroll
                    for (int e = 0; e < kTiles; ++e) o[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    m = -INFINITY;
                    l = 0.0f;
                }
                if (in_use > 0) {
#pragma unroll
                    for (int x = 0; x < B::kLoads; ++x) k_lds[wave][k_slot(row_at + x * kLoadRows, chunk)] = b.k[x];
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
                    if constexpr (kFmt == kFmtFp16) {
#pragma unroll
                        for (int s = 0; s < kSteps; ++s)
                            sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                                __builtin_bit_cast(h16x8, k_lds[wave][k_slot(position(c), 4 * s + j)]), qf[s], sc, 0, 0, 0);
                    } else {
#pragma unroll
                        for (int s = 0; s < kSteps; s += 2) {
                            const Chunk codes = k_lds[wave][k_slot(position(c), 2 * j + s / 2)];
#pragma unroll
                            for (int z = 0; z < 2; ++z) {
                                const h16x8 keys = widen8<kFmt>(codes.w[2 * z], codes.w[2 * z + 1]);
                                sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(keys, qf[s + z], sc, 0, 0, 0);
                            }
                        }
                    }
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    // v4[r]: position(4 j + r), the eight channels (four, 64 channels) of this lane's row of the tiles.
                    h16x8 v4[4];
                    if constexpr (!kNarrow) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) v4[r] = __builtin_bit_cast(h16x8, b.v[r]);
                    } else {
                        // Lanes c and c ^ 8 hold the same chunk of positions 2 j and 2 j + 1 (and 8 more): each keeps one
                        // half of the chunk, the lower lane the lower, and gives away the other.
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            uint32_t keep[2], got[2];
#pragma unroll
                            for (int z = 0; z < 2; ++z) {
                                keep[z] = c < 8 ? b.v[x].w[z] : b.v[x].w[2 + z];
                                got[z] = (uint32_t)__builtin_amdgcn_update_dpp(
                                    0, (int)(c < 8 ? b.v[x].w[2 + z] : b.v[x].w[z]), 0x128, 0xF, 0xF, true);   // row_ror:8
                            }
#pragma unroll
                            for (int odd = 0; odd < 2; ++odd) {
                                const bool own = odd == 0 ? c < 8 : c >= 8;
                                const uint32_t w0 = own ? keep[0] : got[0], w1 = own ? keep[1] : got[1];
                                if constexpr (kFmt == kFmtFp16) v4[2 * x + odd] = __builtin_bit_cast(h16x8, Chunk{{w0, w1, 0, 0}});
                                else v4[2 * x + odd] = widen8<kFmt>(w0, w1);
                            }
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[r] = scaled(sc[r], a.scale_log2);
                    if (in_use < 16) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) sc[r] = position(4 * j + r) < in_use ? sc[r] : -INFINITY;
                    }
                    float mx = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
                    mx = max_xor32(max_xor16(mx));
                    const float m_new = fmaxf(m, mx);
                    const float m_use = m_new == -INFINITY ? 0.0f : m_new;
                    if (__builtin_amdgcn_ballot_w64(m_new > m) != 0) {
                        const float alpha = exp2_fast(m - m_use);
                        l *= alpha;
#pragma unroll
                        for (int e = 0; e < kTiles; ++e)
#pragma unroll
                            for (int r = 0; r < 4; ++r) o[e][r] *= alpha;
                    }
                    m = m_new;
                    h16x4 pf;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float pr = exp2_fast(sc[r] - m_use + kLift);
                        l += pr;
                        pf[r] = (h16)pr;
                    }
#pragma unroll
                    for (int e = 0; e < kTiles; ++e) {
                        // Row n of tile e: channel 8 n + e; of 128-byte rows, channel e of what lane n kept.
                        h16x4 vf;
#pragma unroll
                        for (int r = 0; r < 4; ++r) vf[r] = v4[r][e];
                        o[e] = __builtin_amdgcn_mfma_f32_16x16x16f16(vf, pf, o[e], 0, 0, 0);
                    }
                }
                if (it.meta & kLast) {                     // the waves' states meet in LDS
                    l = sum_xor32(sum_xor16(l));
                    __syncthreads();                       // the last stretch's states have been read
                    if (j == 0) { m_lds[wave][c] = m; l_lds[wave][c] = l; }
                    if (c < heads) {
#pragma unroll
                        for (int e = 0; e < kTiles; ++e)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const int tile_row = 4 * j + r;
                                const int ch = !kNarrow ? 8 * tile_row + e
                                                        : 2 * kTiles * (tile_row & 7) + kTiles * (tile_row >> 3) + e;
                                o_lds[wave][c * kStride + ch] = o[e][r];
                            }
                    }
                    __syncthreads();
                    const int head0 = it.kvh * group + slice * kSliceHeads;
                    const bool whole = (it.meta & kBegun) && (it.meta & kEnded);
                    float* dst = a.parts + (((size_t)worker * 2 + (it.meta & kBegun ? 1 : 0)) * gridDim.y + slice) *
                                               min(group, kSliceHeads) * part_floats(kHd);
                    // Four channels a thread, whole heads side by side; no loop, so that the loads in flight stay so.
                    constexpr int kQuads = kHd / 4, kAtOnce = kBatchThreads / kQuads;
#pragma unroll
                    for (int pass = 0; pass < kSliceHeads / kAtOnce; ++pass) {
                        const int h = tid / kQuads + pass * kAtOnce, ch = 4 * (tid % kQuads);
                        if (h >= heads) continue;
                        float m_all = -INFINITY;
#pragma unroll
                        for (int w = 0; w < kBatchWaves; ++w) m_all = fmaxf(m_all, m_lds[w][h]);
                        f32x4 ov = {0.0f, 0.0f, 0.0f, 0.0f};
                        float l_all = 0.0f;
#pragma unroll
                        for (int w = 0; w < kBatchWaves; ++w) {
                            const float mw = m_lds[w][h];
                            const float f = mw == -INFINITY ? 0.0f : exp2_fast(mw - m_all);
                            const f32x4 ow = *reinterpret_cast<const f32x4*>(&o_lds[w][h * kStride + ch]);
#pragma unroll
                            for (int r = 0; r < 4; ++r) ov[r] = fmaf(ow[r], f, ov[r]);
                            l_all = fmaf(l_lds[w][h], f, l_all);
                        }
                        if (whole) {
                            const float inv = l_all == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(l_all);
                            h16* to = a.out + ((size_t)it.seq * a.n_q_heads + head0 + h) * kHd + ch;
#pragma unroll
                            for (int r = 0; r < 4; ++r) to[r] = to_half(ov[r] * inv);
                        } else {
                            float* rec = dst + (size_t)h * part_floats(kHd);
                            *reinterpret_cast<f32x4*>(rec + ch) = ov;
                            if (ch == 0) { rec[kHd] = m_all; rec[kHd + 1] = l_all; }
                        }
                    }
                }
            };

#pragma unroll
            for (int d = 0; d < kDepth; ++d) fetch(buf[d], qn[d], d);
            for (int i = 0; i < n; i += kDepth) {
#pragma unroll
                for (int d = 0; d < kDepth; ++d) {
                    step(buf[d], qn[d], i + d);
                    fetch(buf[d], qn[d], i + d + kDepth);
                }
            }
            __syncthreads();                               // the items are free again
        }
        chunk_units0 = chunk_units1;
        __syncthreads();
    }
}

// Folds the partial states of the rows that several workers share, in the order of their pages. A workgroup has kHeads
// heads of a row; a thread holds four channels of one of them over every kGroups-th part, and the groups' states meet
// in LDS.
template <int kHd, int kHeads, int kGroups>
__global__ __launch_bounds__(kHd / 4 * kHeads * kGroups) void decode_batch_merge(BatchArgs a, int slices) {
    constexpr int kQuads = kHd / 4;
    __shared__ float s_m[kGroups][kHeads], s_l[kGroups][kHeads];
    __shared__ __attribute__((aligned(16))) float s_o[kGroups > 1 ? kGroups * kHeads * kHd : 1];
    const int group = a.n_q_heads / a.n_kv_heads;
    const int row = (int)blockIdx.x, per = min(group, kSliceHeads);
    const Row at = a.rows[row];
    if (at.first == at.last) return;                                     // that worker wrote the output
    const int quad = (int)threadIdx.x % kQuads, local = (int)threadIdx.x / kQuads % kHeads;
    const int grp = (int)threadIdx.x / (kQuads * kHeads);
    const int want = (int)blockIdx.y * kHeads + local, in_group = min(want, group - 1);
    const int slice = in_group / kSliceHeads, h = in_group - slice * kSliceHeads;
    auto part = [&](int w) {
        return a.parts + ((((size_t)w * 2 + (w == at.first ? 1 : 0)) * slices + slice) * per + h) * part_floats(kHd);
    };
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    constexpr int kAhead = 4;
    for (int w0 = at.first + grp; w0 <= at.last; w0 += kAhead * kGroups) {
        f32x4 ov[kAhead];
        float mv[kAhead], lv[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int w = w0 + i * kGroups;
            const float* p = part(min(w, at.last));
            ov[i] = *reinterpret_cast<const f32x4*>(p + 4 * quad);
            mv[i] = p[kHd];
            lv[i] = w <= at.last ? p[kHd + 1] : 0.0f;      // (behind the last part: the last once more, unused)
        }
        float m_new = m;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) m_new = fmaxf(m_new, mv[i]);
        const float m_use = m_new == -INFINITY ? 0.0f : m_new;
        const float keep = exp2_fast(m - m_use);
        o *= keep;
        l *= keep;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (lv[i] == 0.0f) continue;                   // nothing seen there (a part that saw only NaN has NaN here)
            const float f = exp2_fast(mv[i] - m_use);
            l = fmaf(lv[i], f, l);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = fmaf(ov[i][r], f, o[r]);
        }
        m = m_new;
    }
    if constexpr (kGroups > 1) {
        if (quad == 0) { s_m[grp][local] = m; s_l[grp][local] = l; }
        *reinterpret_cast<f32x4*>(&s_o[(grp * kHeads + local) * kHd + 4 * quad]) = o;
        __syncthreads();
        if (grp > 0) return;
        for (int g = 0; g < kGroups; ++g) m = fmaxf(m, s_m[g][local]);
        const float m_use = m == -INFINITY ? 0.0f : m;
        o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        l = 0.0f;
#pragma unroll 8
        for (int g = 0; g < kGroups; ++g) {
            const float f = exp2_fast(s_m[g][local] - m_use);
            const f32x4 og = *reinterpret_cast<const f32x4*>(&s_o[(g * kHeads + local) * kHd + 4 * quad]);
            l = fmaf(s_l[g][local], f, l);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = fmaf(og[r], f, o[r]);
        }
    }
    if (want >= group) return;
    const int seq = row / a.n_kv_heads, kvh = row - seq * a.n_kv_heads;
    h16* dst = a.out + ((size_t)seq * a.n_q_heads + kvh * group + in_group) * kHd + 4 * quad;
    const float inv = l == 0.0f ? 0.0f : __builtin_amdgcn_rcpf(l);      // 1 ulp of FP32
#pragma unroll
    for (int r = 0; r < 4; ++r) dst[r] = to_half(o[r] * inv);
}

// Any head_dim <= 256, any alignment, FP16: a wave per (sequence, head) walks the sequence's keys.
__global__ __launch_bounds__(kWave) void decode_batch_generic(BatchArgs a, int head_dim) {
    const int seq = (int)blockIdx.x, head = (int)blockIdx.y, lane = lane_id();
    const int kvh = head / (a.n_q_heads / a.n_kv_heads);
    const int len = seen_len(a, seq);
    const int* table = a.tables + (size_t)seq * a.max_pages;
    const h16* q = a.q + ((size_t)seq * a.n_q_heads + head) * head_dim;
    float qv[4], acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        qv[i] = d < head_dim ? (float)q[d] : 0.0f;
        acc[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int t = 0; t < len; ++t) {
        const int page = table[t / kPage];
        if (page < 0 || page >= a.n_pages) continue;
        const size_t at = (((size_t)page * kPage + t % kPage) * a.n_kv_heads + kvh) * head_dim;
        const h16* k = static_cast<const h16*>(a.k) + at;
        const h16* v = static_cast<const h16*>(a.v) + at;
        float dot = 0.0f, vv4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 64 * i;
            dot = d < head_dim ? fmaf(qv[i], (float)k[d], dot) : dot;
            vv4[i] = d < head_dim ? (float)v[d] : 0.0f;
        }
        const float s = scaled(wave_sum(dot), a.scale_log2);
        const float m_new = fmaxf(m, s), m_use = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = exp2_fast(m - m_use), p = exp2_fast(s - m_use);
        m = m_new;
        l = fmaf(l, alpha, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(acc[i], alpha, p * vv4[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        if (d < head_dim)
            a.out[((size_t)seq * a.n_q_heads + head) * head_dim + d] = to_half(l == 0.0f ? 0.0f : acc[i] / l);
    }
}

inline size_t row_bytes(int n_seqs, int n_kv_heads) {
    return ((size_t)n_seqs * n_kv_heads * sizeof(Row) + 255) & ~(size_t)255;
}

template <int kHd, int kFmt>
void launch(const BatchArgs& a, int slices, hipStream_t st) {
    decode_batch<kHd, kFmt><<<dim3(kWorkers, (unsigned)slices), kBatchThreads, 0, st>>>(a);
}

template <int kHd, int kHeads, int kThreads>
void launch_merge_of(const BatchArgs& a, int slices, hipStream_t st) {
    const dim3 grid((unsigned)(a.n_seqs * a.n_kv_heads), (unsigned)((a.n_q_heads / a.n_kv_heads - 1) / kHeads + 1));
    decode_batch_merge<kHd, kHeads, kThreads * 4 / (kHd * kHeads)><<<grid, kThreads, 0, st>>>(a, slices);
}
// The fewer rows, the more parts a row can have, and the more threads are put to one; but a workgroup costs its launch
// also where a row has nothing to fold, which is what many rows mostly have. Measured (both launches) at 28 + 4 heads with
// one head of 1024 threads / one of 256 / two of 256 / four of 256 / eight of 256 a workgroup, in us:
//   one sequence of 14449 positions (4 rows)             14.8 / 16.3 / 19.9 / 27.9 / 43.5
//   8 of 2048 (32 rows)                                  14.6 / 13.8 / 13.8 / 14.5 / 15.8
//   one of 14449 and 39 of 60 (160 rows)                 18.2 / 18.0 / 20.9 / 26.2 / 36.3
//   128 of 50 .. 150 (512 rows)                          20.0 / 14.8 / 14.6 / 14.6 / 14.1
//   one of 32000 and 249 of 60 (1000 rows)               34.7 / 31.1 / 32.6 / 36.1 / 43.8
//   1000 of 64 (4000 rows)                               57.8 / 40.1 / 37.7 / 36.0 / 35.2
template <int kHd>
void launch_merge(const BatchArgs& a, int slices, hipStream_t st) {
    const int rows = a.n_seqs * a.n_kv_heads;
    if (rows <= 16) launch_merge_of<kHd, 1, 1024>(a, slices, st);
    else if (rows <= 1024) launch_merge_of<kHd, 1, 256>(a, slices, st);
    else launch_merge_of<kHd, 4, 256>(a, slices, st);
}

}  // namespace
}  // namespace vv

extern "C" {

size_t vv_attn_decode_batch_scratch_bytes(int n_seqs, int n_q_heads, int n_kv_heads, int head_dim) {
    if (n_seqs <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || n_q_heads % n_kv_heads) return 0;
    const int group = n_q_heads / n_kv_heads, slices = (group + vv::kSliceHeads - 1) / vv::kSliceHeads;
    return vv::row_bytes(n_seqs, n_kv_heads) + (size_t)vv::kWorkers * 2 * slices * std::min(group, vv::kSliceHeads) *
                                                   vv::part_floats(head_dim) * sizeof(float);
}

vv_status_t vv_attn_decode_batch(int backend, const void* q, const vv_kv_view_t* kv, void* out, int n_q_heads,
                                 int n_seqs, const int* cache_lens, int max_pages, int n_pages, void* scratch,
                                 size_t scratch_bytes, void* stream) {
    (void)backend;
    if (!q || !kv || !out || !cache_lens) return VV_ERR_NULL_PTR;
    if (n_seqs <= 0) return VV_OK;
    if (!kv->k || !kv->v || !kv->page_table) return VV_ERR_NULL_PTR;
    const bool fp8 = kv->format == vv::kFmtE4M3 || kv->format == vv::kFmtE5M2;
    if (kv->format != vv::kFmtFp16 && !(fp8 && kv->head_dim == 128)) return VV_ERR_UNSUPPORTED;
    if (n_q_heads <= 0 || n_q_heads > (1 << 14) || kv->n_kv_heads <= 0 || n_q_heads % kv->n_kv_heads ||
        kv->head_dim <= 0 || kv->head_dim > 256)
        return VV_ERR_UNSUPPORTED;
    if (max_pages <= 0 || n_pages <= 0) return VV_ERR_INVALID_ARG;
    // the list of (sequence, KV head, page) is counted in 32 bits, and a launch has a workgroup per row of it
    if ((int64_t)n_seqs * kv->n_kv_heads > (1 << 22) || (int64_t)max_pages * vv::kPage > INT32_MAX ||
        (int64_t)n_seqs * max_pages * kv->n_kv_heads > INT32_MAX - vv::kWorkers)
        return VV_ERR_UNSUPPORTED;
    vv::BatchArgs a = {static_cast<const vv::h16*>(q), kv->k, kv->v, kv->page_table, cache_lens,
                       static_cast<vv::h16*>(out), nullptr, nullptr, n_q_heads, kv->n_kv_heads, n_seqs, max_pages,
                       n_pages, vv::kLog2e / sqrtf((float)kv->head_dim)};
    hipStream_t st = vv::as_stream(stream);
    const bool aligned = vv::aligned16(q) && vv::aligned16(kv->k) && vv::aligned16(kv->v);
    if (fp8 && !aligned) return VV_ERR_UNSUPPORTED;
    if (aligned && (kv->head_dim == 128 || kv->head_dim == 64)) {
        const size_t want = vv_attn_decode_batch_scratch_bytes(n_seqs, n_q_heads, kv->n_kv_heads, kv->head_dim);
        if (!scratch) return VV_ERR_NULL_PTR;
        if (scratch_bytes < want || !vv::aligned16(scratch)) return VV_ERR_INVALID_ARG;
        a.rows = static_cast<vv::Row*>(scratch);
        a.parts = reinterpret_cast<float*>(static_cast<char*>(scratch) + vv::row_bytes(n_seqs, kv->n_kv_heads));
        const int group = n_q_heads / kv->n_kv_heads, slices = (group + vv::kSliceHeads - 1) / vv::kSliceHeads;
        if (kv->head_dim == 64) vv::launch<64, vv::kFmtFp16>(a, slices, st);
        else if (kv->format == vv::kFmtFp16) vv::launch<128, vv::kFmtFp16>(a, slices, st);
        else if (kv->format == vv::kFmtE4M3) vv::launch<128, vv::kFmtE4M3>(a, slices, st);
        else vv::launch<128, vv::kFmtE5M2>(a, slices, st);
        if (hipGetLastError() != hipSuccess) return VV_ERR_CUDA_LAUNCH;
        if (kv->head_dim == 64) vv::launch_merge<64>(a, slices, st);
        else vv::launch_merge<128>(a, slices, st);
    } else {
        const dim3 grid((unsigned)n_seqs, (unsigned)n_q_heads);
        vv::decode_batch_generic<<<grid, vv::kWave, 0, st>>>(a, kv->head_dim);
    }
    return vv::launch_status();
}

}  // extern "C"
