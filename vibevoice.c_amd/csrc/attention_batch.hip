// Decode attention of many sequences over one paged pool: one query row per sequence and head, each sequence behind its
// own row of page ids and of its own length, the lengths on the device.
#include <algorithm>

#include "attn_common.hpp"

namespace vv {
namespace {

constexpr int kBatchThreads = 256;
constexpr int kBatchWaves = kBatchThreads / kWave;
constexpr int kWorkers = 1024;
constexpr int kSliceHeads = 16;              // query heads of a group that one workgroup takes: a matrix tile's columns

struct BatchArgs {
    const h16* q;
    const void* k;
    const void* v;
    const int* tables;
    const int* lens;
    h16* out;
    int* starts;            // [n_seqs + 1] pages before each sequence
    float* parts;
    int n_q_heads, n_kv_heads, n_seqs, max_pages, n_pages;
    float scale_log2;
};

__device__ __forceinline__ int seen_len(const BatchArgs& a, int s) { return min(max(a.lens[s], 0), a.max_pages * kPage); }
__device__ __forceinline__ int pages_of(int len) { return (len + kPage - 1) / kPage; }

__device__ __forceinline__ int wave_prefix(int v) {       // inclusive
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
        const int o = __shfl_up(v, d);
        if (lane_id() >= d) v += o;
    }
    return v;
}

// A worker's units: [first, last) of the row-major list (sequence, KV head, page).
__device__ __forceinline__ int units_each(int units) { return (units + kWorkers - 1) / kWorkers; }

// Where a worker leaves the partial state of a stretch: rows that begin inside the worker and run on, or ran on into it.
__device__ __forceinline__ size_t part_floats(int group_heads, int hd) { return (size_t)group_heads * (hd + 4); }

template <int kHd, int kFmt>
struct Blocks {             // a wave's sixteen keys as they were loaded
    static constexpr int kUnit = kFmt == kFmtFp16 ? 2 : 1;
    static constexpr int kRow = kHd * kUnit;              // bytes per vector
    static constexpr int kKLoads = kRow / 64;             // 16-byte loads of K per lane
    Chunk k[kKLoads];
    Chunk v[4];             // FP8: the lower eight bytes
};

template <int kHd, int kFmt>
__global__ __launch_bounds__(kBatchThreads, 4) void decode_batch(BatchArgs a) {
    typedef Blocks<kHd, kFmt> B;
    constexpr int kSteps = kHd / 32;                       // 32-channel steps of the score product
    constexpr int kChunks = kHd / 8;
    constexpr int kTiles = kHd / 16;                       // O^T tiles
    constexpr int kStride = kHd + 1;
    __shared__ float o_lds[kBatchWaves][kSliceHeads * kStride];
    __shared__ float m_lds[kBatchWaves][16], l_lds[kBatchWaves][16];
    __shared__ int s_sum[kBatchWaves], s_at[3];

    const int tid = (int)threadIdx.x, lane = tid & 63, wave = wave_in_block();
    const int c = lane & 15, j = lane >> 4;
    const int worker = (int)blockIdx.x, slice = (int)blockIdx.y;
    const int group = a.n_q_heads / a.n_kv_heads;
    const int heads = min(kSliceHeads, group - slice * kSliceHeads);      // of this slice

    // Pages before every sequence.
    const int each = (a.n_seqs + kBatchThreads - 1) / kBatchThreads;
    int mine = 0;
    for (int i = 0; i < each; ++i) {
        const int s = tid * each + i;
        if (s < a.n_seqs) mine += pages_of(seen_len(a, s));
    }
    const int incl = wave_prefix(mine);
    if (lane == 63) s_sum[wave] = incl;
    if (tid == 0) { s_at[0] = a.n_seqs; s_at[1] = 0; }
    __syncthreads();
    int before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kBatchWaves; ++w) {
        if (w < wave) before += s_sum[w];
        total += s_sum[w];
    }
    const int units = total * a.n_kv_heads, per = units_each(units);
    int u = min(worker * per, units);
    const int u_end = min(u + per, units);
    if (worker == 0 && slice == 0) {
        int at = before;
        for (int i = 0; i < each; ++i) {
            const int s = tid * each + i;
            if (s < a.n_seqs) {
                a.starts[s] = at;
                at += pages_of(seen_len(a, s));
            }
        }
        if (tid == 0) a.starts[a.n_seqs] = total;
    }
    // Sequences without positions: zeros.
    for (int s = worker; s < a.n_seqs; s += kWorkers) {
        if (seen_len(a, s) > 0) continue;
        for (int i = tid; i < heads * a.n_kv_heads * kHd; i += kBatchThreads) {
            const int kvh = i / (heads * kHd), e = i - kvh * heads * kHd;
            a.out[((size_t)s * a.n_q_heads + kvh * group + slice * kSliceHeads) * kHd + e] = (h16)0.0f;
        }
    }
    if (u >= u_end) return;
    // The sequence the first unit lies in.
    {
        int at = before;
        for (int i = 0; i < each; ++i) {
            const int s = tid * each + i;
            const int n = s < a.n_seqs ? pages_of(seen_len(a, s)) : 0;
            if (n > 0 && at * a.n_kv_heads <= u && u < (at + n) * a.n_kv_heads) {
                s_at[0] = s;
                s_at[1] = at;
            }
            at += n;
        }
    }
    __syncthreads();
    int seq = s_at[0], unit0 = s_at[1] * a.n_kv_heads;     // its first unit

    while (u < u_end && seq < a.n_seqs) {
        const int len = seen_len(a, seq), n_pages = pages_of(len);
        if (n_pages == 0) { ++seq; continue; }
        const int kvh = (u - unit0) / n_pages, page0 = (u - unit0) - kvh * n_pages;
        const int page1 = min(n_pages, page0 + (u_end - u));
        const int* table = a.tables + (size_t)seq * a.max_pages;
        const size_t row_bytes = (size_t)a.n_kv_heads * B::kRow;

        const int head0 = kvh * group + slice * kSliceHeads;
        h16x8 qf[kSteps];
        {
            const Chunk* qp = reinterpret_cast<const Chunk*>(a.q + ((size_t)seq * a.n_q_heads + head0 + min(c, heads - 1)) * kHd);
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
                qf[s] = __builtin_bit_cast(h16x8, load_chunk(qp + (kFmt == kFmtFp16 ? 4 * s + j : 4 * j + s)));
        }
        f32x4 o[kTiles];
#pragma unroll
        for (int e = 0; e < kTiles; ++e) o[e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;

        for (int p = page0; p < page1; ++p) {
            const int key0 = p * kPage + 16 * wave;        // this wave's sixteen keys
            const int page = __builtin_amdgcn_readfirstlane(table[p]);
            const bool bad = page < 0 || page >= a.n_pages;
            if (key0 >= len || bad) continue;
            const char* kp = static_cast<const char*>(a.k) + ((size_t)page * kPage + 16 * wave) * row_bytes + (size_t)kvh * B::kRow;
            const char* vp = static_cast<const char*>(a.v) + ((size_t)page * kPage + 16 * wave) * row_bytes + (size_t)kvh * B::kRow;
            B b;
#pragma unroll
            for (int i = 0; i < B::kKLoads; ++i) {
                const int at = kFmt == kFmtFp16 ? 64 * i + 16 * j : 32 * j + 16 * i;
                b.k[i] = load_chunk_stream(reinterpret_cast<const Chunk*>(kp + c * row_bytes + at));
            }
            h16x8 v4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const char* at = vp + (4 * j + i) * row_bytes + (c % kChunks) * (8 * B::kUnit);
                if constexpr (kFmt == kFmtFp16) {
                    v4[i] = __builtin_bit_cast(h16x8, load_chunk_stream(reinterpret_cast<const Chunk*>(at)));
                } else {
                    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
                    const u32x2 codes = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(at));
                    Chunk w;
                    widen4<kFmt>(codes.x, w.w[0], w.w[1]);
                    widen4<kFmt>(codes.y, w.w[2], w.w[3]);
                    v4[i] = __builtin_bit_cast(h16x8, w);
                }
            }
            f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                Chunk w;
                if constexpr (kFmt == kFmtFp16) {
                    w = b.k[s];
                } else {
                    widen4<kFmt>(b.k[s / 2].w[2 * (s & 1)], w.w[0], w.w[1]);
                    widen4<kFmt>(b.k[s / 2].w[2 * (s & 1) + 1], w.w[2], w.w[3]);
                }
                sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, w), qf[s], sc, 0, 0, 0);
            }
            if (key0 + 16 > len) {                         // what lies past the end is masked, whatever it holds
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool in = key0 + 4 * j + r < len;
                    sc[r] = in ? sc[r] : -INFINITY;
                    if (!in) v4[r] = h16x8{0, 0, 0, 0, 0, 0, 0, 0};
                }
            }
            float mx = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
            mx = max_xor32(max_xor16(mx)) * a.scale_log2;
            const float m_new = fmaxf(m, mx);
            const float m_use = m_new == -INFINITY ? 0.0f : m_new;
            const float alpha = exp2_fast(m - m_use);
            l *= alpha;
#pragma unroll
            for (int e = 0; e < kTiles; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[e][r] *= alpha;
            m = m_new;
            h16x4 pf;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float pr = exp2_fast(fmaf(sc[r], a.scale_log2, -m_use));
                l += pr;
                pf[r] = (h16)pr;
            }
#pragma unroll
            for (int e = 0; e < kTiles; ++e) {
                // 128 channels: tile e is the channels 8 c + e. 64: chunk c % 8's channel e + 4 (c / 8).
                h16x4 vf;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (kChunks == 16) vf[r] = v4[r][e];
                    else vf[r] = c < 8 ? v4[r][e] : v4[r][e + 4];
                }
                o[e] = __builtin_amdgcn_mfma_f32_16x16x16f16(vf, pf, o[e], 0, 0, 0);
            }
        }

        // The waves' states meet in LDS.
        l = sum_xor32(sum_xor16(l));
        __syncthreads();
        if (j == 0) { m_lds[wave][c] = m; l_lds[wave][c] = l; }
        if (c < heads) {
#pragma unroll
            for (int e = 0; e < kTiles; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int tile_row = 4 * j + r;
                    const int ch = kChunks == 16 ? 8 * tile_row + e : 8 * (tile_row & 7) + e + 4 * (tile_row >> 3);
                    o_lds[wave][c * kStride + ch] = o[e][r];
                }
        }
        __syncthreads();
        const bool whole = page0 == 0 && page1 == n_pages;
        float* dst = a.parts + (((size_t)worker * 2 + (page0 == 0 ? 1 : 0)) * gridDim.y + slice) *
                                   part_floats(min(group, kSliceHeads), kHd);
        for (int i = tid; i < heads * kHd; i += kBatchThreads) {
            const int h = i / kHd, ch = i % kHd;
            float m_all = -INFINITY;
#pragma unroll
            for (int w = 0; w < kBatchWaves; ++w) m_all = fmaxf(m_all, m_lds[w][h]);
            float ov = 0.0f, l_all = 0.0f;
#pragma unroll
            for (int w = 0; w < kBatchWaves; ++w) {
                const float mw = m_lds[w][h];
                const float f = mw == -INFINITY ? 0.0f : exp2_fast(mw - m_all);
                ov = fmaf(o_lds[w][h * kStride + ch], f, ov);
                l_all = fmaf(l_lds[w][h], f, l_all);
            }
            if (whole) {
                a.out[((size_t)seq * a.n_q_heads + head0 + h) * kHd + ch] = to_half(l_all == 0.0f ? 0.0f : ov / l_all);
            } else {
                float* rec = dst + (size_t)h * (kHd + 4);
                rec[ch] = ov;
                if (ch == 0) { rec[kHd] = m_all; rec[kHd + 1] = l_all; }
            }
        }
        u += page1 - page0;
        if (u == unit0 + n_pages * a.n_kv_heads) { ++seq; unit0 = u; }
    }
}

// Folds the stretches of a row (sequence, KV head) that several workers share.
template <int kHd>
__global__ __launch_bounds__(256) void decode_batch_merge(BatchArgs a, int slices) {
    const int group = a.n_q_heads / a.n_kv_heads;
    const int seq = (int)blockIdx.x, head = (int)blockIdx.y, kvh = head / group, in_group = head - kvh * group;
    const int slice = in_group / kSliceHeads, h = in_group - slice * kSliceHeads;
    const int total = a.starts[a.n_seqs] * a.n_kv_heads, per = units_each(total);
    const int pages = a.starts[seq + 1] - a.starts[seq];
    if (pages == 0) return;
    const int u0 = a.starts[seq] * a.n_kv_heads + kvh * pages, u1 = u0 + pages;
    const int first = u0 / per, last = (u1 - 1) / per;
    if (first == last) return;                                     // that worker wrote the output
    const size_t record = part_floats(min(group, kSliceHeads), kHd);
    auto part = [&](int w) {
        return a.parts + (((size_t)w * 2 + (w == first ? 1 : 0)) * slices + slice) * record + (size_t)h * (kHd + 4);
    };
    const int ch = (int)threadIdx.x;
    if (ch >= kHd) return;
    float m_all = -INFINITY;
    for (int w = first; w <= last; ++w) m_all = fmaxf(m_all, part(w)[kHd]);
    float o = 0.0f, l = 0.0f;
    for (int w = first; w <= last; ++w) {
        const float* p = part(w);
        const float f = p[kHd] == -INFINITY ? 0.0f : exp2_fast(p[kHd] - m_all);
        o = fmaf(p[ch], f, o);
        l = fmaf(p[kHd + 1], f, l);
    }
    a.out[((size_t)seq * a.n_q_heads + head) * kHd + ch] = to_half(l == 0.0f ? 0.0f : o / l);
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
        const float s = wave_sum(dot) * a.scale_log2;
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

inline size_t starts_bytes(int n_seqs) { return (((size_t)n_seqs + 1) * sizeof(int) + 255) & ~(size_t)255; }

}  // namespace
}  // namespace vv

extern "C" {

size_t vv_attn_decode_batch_scratch_bytes(int n_seqs, int n_q_heads, int n_kv_heads, int head_dim) {
    if (n_seqs <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || n_q_heads % n_kv_heads) return 0;
    const int group = n_q_heads / n_kv_heads, slices = (group + vv::kSliceHeads - 1) / vv::kSliceHeads;
    return vv::starts_bytes(n_seqs) + (size_t)vv::kWorkers * 2 * slices * std::min(group, vv::kSliceHeads) *
                                          ((size_t)head_dim + 4) * sizeof(float);
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
    if (n_q_heads <= 0 || kv->n_kv_heads <= 0 || n_q_heads % kv->n_kv_heads || kv->head_dim <= 0 || kv->head_dim > 256)
        return VV_ERR_UNSUPPORTED;
    if (max_pages <= 0 || n_pages <= 0) return VV_ERR_INVALID_ARG;
    // the list of (sequence, KV head, page) is counted in 32 bits
    if ((int64_t)max_pages * vv::kPage > INT32_MAX || (int64_t)n_seqs * max_pages * kv->n_kv_heads > INT32_MAX - vv::kWorkers)
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
        a.starts = static_cast<int*>(scratch);
        a.parts = reinterpret_cast<float*>(static_cast<char*>(scratch) + vv::starts_bytes(n_seqs));
        const int group = n_q_heads / kv->n_kv_heads, slices = (group + vv::kSliceHeads - 1) / vv::kSliceHeads;
        const dim3 grid(vv::kWorkers, (unsigned)slices), merge((unsigned)n_seqs, (unsigned)n_q_heads);
        if (kv->head_dim == 64)
            vv::decode_batch<64, vv::kFmtFp16><<<grid, vv::kBatchThreads, 0, st>>>(a);
        else if (kv->format == vv::kFmtFp16)
            vv::decode_batch<128, vv::kFmtFp16><<<grid, vv::kBatchThreads, 0, st>>>(a);
        else if (kv->format == vv::kFmtE4M3)
            vv::decode_batch<128, vv::kFmtE4M3><<<grid, vv::kBatchThreads, 0, st>>>(a);
        else
            vv::decode_batch<128, vv::kFmtE5M2><<<grid, vv::kBatchThreads, 0, st>>>(a);
        if (hipGetLastError() != hipSuccess) return VV_ERR_CUDA_LAUNCH;
        if (kv->head_dim == 64)
            vv::decode_batch_merge<64><<<merge, 64, 0, st>>>(a, slices);
        else
            vv::decode_batch_merge<128><<<merge, 128, 0, st>>>(a, slices);
    } else {
        const dim3 grid((unsigned)n_seqs, (unsigned)n_q_heads);
        vv::decode_batch_generic<<<grid, vv::kWave, 0, st>>>(a, kv->head_dim);
    }
    return vv::launch_status();
}

}  // extern "C"
