// The cache side of a serving step: many sequences that share one pool of 64-position pages.
//
//   page_plan       which pages and slots a step's new positions take, from the sequences' lengths.
//   append_rows     bias, rotary embedding and the append of a step's rows, each at its own position and slot.
//
// Both are described at their kernels; the attention that reads the pool is in attention_batch.hip.
#include "attn_common.hpp"
#include "rope_common.hpp"

namespace vv {
namespace {

// ── pages and slots from lengths ─────────────────────────────────────────
// Sequence i holds len_i positions and asks for new_i more: need_i = ceil((len_i + new_i) / 64) - ceil(len_i / 64)
// pages. Sequences are served in order: with E_i the running sum of new rows and C_i that of needed pages (both
// through i), i is served when its positions fit its table, its rows end within max_rows (E_i <= max_rows) and it
// needs no page or C_i <= n_free. C counts a sequence that is turned away for want of pages too, so none that needs
// a page overtakes it, and the served ones' pages are the first C of the stack, without holes:
// page j handed out is free[n_free - 1 - j].
// Everything a row writes follows from its own sequence's E, C and length, so every workgroup scans the lengths for
// itself (8 bytes a sequence, out of L2) and fills its own run of rows: one launch, no exchange between workgroups,
// no atomics on memory. A new page's first position is always a new row, so that row writes the table entry.
// Sums are 32 bits, held at 2^31 - 1: past that no row or page is handed out, and the saturating sum of
// non-negative values does not depend on its grouping.
struct PlanArgs {
    const int* new_lens;
    const int* cache_lens;
    int* tables;
    const int* free_pages;
    const int* n_free;
    int* lens_out;
    int* row_starts;
    int* positions;
    int64_t* slots;
    int* n_free_out;         // or nullptr
    int* counts;
    int n_seqs, max_pages, max_rows, rows_per_wg;
};

constexpr int kPlanThreads = 1024;

__device__ __forceinline__ int add_capped(int a, int b) {
    const uint32_t s = (uint32_t)a + (uint32_t)b;
    return s > 0x7fffffffu ? 0x7fffffff : (int)s;
}

template <int kCtrl, int kRows>
__device__ __forceinline__ int scan_step(int v) {
    return add_capped(v, __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xF, false));
}
// Inclusive sum over the wave's lanes, inside the vector ALU: shifts by 1, 2, 4, 8 within rows of 16 lanes, then the
// last lane of a row into the next row, then of the first half into the second.
__device__ __forceinline__ int wave_scan(int v) {
    v = scan_step<0x111, 0xF>(v);
    v = scan_step<0x112, 0xF>(v);
    v = scan_step<0x114, 0xF>(v);
    v = scan_step<0x118, 0xF>(v);
    v = scan_step<0x142, 0xA>(v);
    return scan_step<0x143, 0xC>(v);
}
// Inclusive sum over the workgroup and, in `total`, the sum of all; `sums` (an int per wave) is free again after the
// caller's next barrier.
__device__ __forceinline__ int block_scan(int v, int* sums, int& total) {
    const int incl = wave_scan(v);
    const int wave = wave_in_block(), waves = (int)blockDim.x >> 6;
    if (lane_id() == 63) sums[wave] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < waves; ++w) {
        if (w == wave) before = total;
        total = add_capped(total, sums[w]);
    }
    return add_capped(before, incl);
}

__device__ __forceinline__ int pages_of(int len) { return (int)(((unsigned)len + (kPage - 1)) / kPage); }

__global__ __launch_bounds__(kPlanThreads) void page_plan(PlanArgs a) {
    __shared__ int s_rows[kPlanThreads / kWave], s_pages[kPlanThreads / kWave];
    __shared__ int s_end[kPlanThreads], s_start[kPlanThreads], s_len[kPlanThreads], s_fresh[kPlanThreads];
    __shared__ int s_asked, s_given, s_refused;
    const int tid = (int)threadIdx.x, threads = (int)blockDim.x;
    const bool lead = blockIdx.x == 0;           // writes what there is one of: the lengths, row starts and counts
    const int row0 = (int)min((int64_t)blockIdx.x * a.rows_per_wg, (int64_t)a.max_rows);
    const int row1 = (int)min((int64_t)row0 + a.rows_per_wg, (int64_t)a.max_rows);
    const int n_free = max(*a.n_free, 0);
    if (tid == 0) { s_asked = 0; s_given = 0; s_refused = 0; }

    int rows_before = 0, pages_before = 0;
    for (int c0 = 0; c0 < a.n_seqs; c0 += threads) {
        const int i = c0 + tid;
        const int asked = i < a.n_seqs ? max(a.new_lens[i], 0) : 0;
        const int len = i < a.n_seqs ? a.cache_lens[i] : 0;
        int rows_here, pages_here;
        const int end = add_capped(rows_before, block_scan(asked, s_rows, rows_here));
        const bool fits = asked > 0 && len >= 0 && (int64_t)len + asked <= (int64_t)a.max_pages * kPage &&
                          end <= a.max_rows;
        const int need = fits ? pages_of(len + asked) - pages_of(len) : 0;
        const int taken = add_capped(pages_before, block_scan(need, s_pages, pages_here));
        const bool served = fits && (need == 0 || taken <= n_free);
        s_end[tid] = end;
        s_start[tid] = end - asked;
        s_len[tid] = served ? len : -1;
        s_fresh[tid] = taken - need;
        if (lead && i < a.n_seqs) {
            a.lens_out[i] = len + (served ? asked : 0);
            a.row_starts[i + 1] = min(end, a.max_rows);
            if (served) atomicMax(&s_asked, taken);
            if (served && need > 0) atomicMax(&s_given, taken);
            if (asked > 0 && !served) atomicAdd(&s_refused, 1);
        }
        __syncthreads();
        const int rows_after = add_capped(rows_before, rows_here);
        // Unsigned: a saturated sum plus a thread's number stays below 2^32.
        for (unsigned r = (unsigned)max(row0, rows_before) + tid; r < (unsigned)min(row1, rows_after); r += threads) {
            int lo = 0, hi = threads - 1;        // the first sequence of this run that ends past row r
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (s_end[mid] > (int)r) hi = mid;
                else lo = mid + 1;
            }
            const int held = s_len[lo];
            int position = 0;
            int64_t slot = -1;
            if (held >= 0) {
                position = held + ((int)r - s_start[lo]);
                const int index = position / kPage, had = pages_of(held);
                int* entry = a.tables + (size_t)(c0 + lo) * a.max_pages + index;
                int page;
                if (index < had) {
                    page = *entry;
                } else {
                    page = a.free_pages[n_free - 1 - (s_fresh[lo] + index - had)];
                    if (position % kPage == 0) *entry = page;
                }
                if (page >= 0) slot = (int64_t)page * kPage + position % kPage;
            }
            a.positions[r] = position;
            a.slots[r] = slot;
        }
        rows_before = rows_after;
        pages_before = add_capped(pages_before, pages_here);
        __syncthreads();
        if (!lead && rows_before >= row1) return;      // the same for the whole workgroup
    }
    for (unsigned r = (unsigned)max(row0, rows_before) + tid; r < (unsigned)row1; r += threads) {      // rows past the last
        a.positions[r] = 0;
        a.slots[r] = -1;
    }
    if (lead && tid == 0) {
        a.row_starts[0] = 0;
        if (a.n_free_out) *a.n_free_out = n_free - s_given;
        a.counts[0] = n_free - s_asked;
        a.counts[1] = min(rows_before, a.max_rows);
        a.counts[2] = s_refused;
    }
}

// ── bias, rotation and append ────────────────────────────────────────────
// Row r: q_out[r] = rope(q[r] + bq), K[slot_r] = rope(k[r] + bk), V[slot_r] = v[r] + bv at position pos_r, in FP32 with
// one rounding to FP16 (a biased value is not rounded before it is turned: separate calls, which store it there, are
// off by sqrt(2) as much). The angle and the rotation are those of vv_rope_dev, and an FP8 code is that of the
// FP16 value, so without biases the bits are those of vv_rope_qk_dev and vv_kv_store_dev on that row. A row moves
// 4 hd (nq + nkv) + 2 hd nkv b bytes, b the bytes of a stored value, and does three flops a value: bound by memory, or
// by its latency when there are few rows.
// A thread's item is one pair of chunks (c, c + hd/16) of one head: the eight rotary pairs (d, d + hd/2), or for V just
// sixteen values. Heads are counted q, then k, then v. A workgroup owns whole rows, one where a row has 128 items or
// more: its threads ask for their items first, then compute the row's cosines and sines, one pair a thread, into LDS
// under the loads, and rotate and store behind one barrier. The one-row kernel stores non-temporally in launches of 2 MiB
// and more (14449 rows: 45.8 us, 50.5 without) but loads ordinarily: q, k and v were just written by the projections, and
// what of them is still cached is worth more than the hint (4096 rows: 12.5 us, 14.9 with it; 14449 rows 45.8 and 45.1).
// The kernel of short and of very long rows stores ordinarily at every size: at 14 + 2 heads of 64 with the hint, 1000 to
// 4096 rows are the same, 14449 rows 14.4 us instead of 13.6, and launches past 250 MB gain (60000 rows 55.9 instead of
// 60.4; 4000 rows of 100 + 16 heads of 128 50.0 instead of 54.7). Measured at 28 + 4 heads of 128 with
// biases: 16 rows 3.0 us, 2161 rows into an E4M3 pool 8.6, 4096 rows 12.5 (6.0 TB/s), 14449 rows 46 us (5.8 TB/s), into
// an E4M3 pool 45.6.
struct AppendArgs {
    const h16* q;
    const h16* k;
    const h16* v;
    const h16* q_bias;
    const h16* k_bias;
    const h16* v_bias;
    const int* positions;
    const int64_t* slots;
    h16* q_out;
    void* k_store;
    void* v_store;
    int64_t n_slots;
    int rows, nq, nkv, head_dim;
};

// fp8_encode of a value that is an FP16 value already, without branches, on its bits. E5M2 is the top byte of FP16 and
// E4M3 its exponent less 8 with three bits of mantissa, so from the smallest normal on a code is those bits rounded to
// nearest even (a carry runs into the exponent by itself), held at the largest finite one; below, it is the count of
// subnormal steps rounded half up. NaN gives a signed zero.
template <bool kE5M2>
__device__ __forceinline__ uint32_t fp8_code(h16 v) {
    const uint32_t bits = __builtin_bit_cast(uint16_t, v), mag = bits & 0x7FFFu;
    uint32_t code;
    if constexpr (kE5M2) {
        code = (mag + (mag < 0x400u ? 0x80u : 0x7Fu + ((mag >> 8) & 1u))) >> 8;
        code = min(code, 0x7Bu);
    } else {
        const uint32_t low = (uint32_t)fmaf(fabsf((float)v), 512.0f, 0.5f);
        code = (mag - 0x2000u + 0x3Fu + ((mag >> 7) & 1u)) >> 7;
        code = mag < 0x2400u ? low : min(code, 0x7Eu);
    }
    return ((bits >> 8) & 0x80u) | (mag > 0x7C00u ? 0u : code);
}

template <int kFmt, bool kStream>
__device__ __forceinline__ void store_values(void* store, size_t at, const Chunk& c) {      // eight, at element `at`
    if constexpr (kFmt == kFmtFp16) {
        store_chunk_as<kStream>(reinterpret_cast<Chunk*>(static_cast<h16*>(store) + at), c);
    } else {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const h16x8 h = __builtin_bit_cast(h16x8, c);
        u32x2 w = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i >> 2] |= fp8_code<kFmt == kFmtE5M2>(h[i]) << (8 * (i & 3));
        u32x2* dst = reinterpret_cast<u32x2*>(static_cast<uint8_t*>(store) + at);
        if constexpr (kStream) __builtin_nontemporal_store(w, dst);
        else *dst = w;
    }
}

constexpr int kAppendThreads = 1024;      // at most
constexpr int kAppendRows = 8;            // rows a workgroup owns, at most

// (These take the arguments by value: behind a reference, a choice between two of them becomes a choice between two
// addresses, and the compiler keeps the struct in scratch memory - 181 us instead of 46 at 14449 rows.)
// What a thread does with its item once everything has arrived: bias, rotation, one rounding, the stores.
template <int kHd, int kFmt, bool kStream>
__device__ __forceinline__ void finish_item(AppendArgs a, size_t row, int64_t slot, int kind, int h, int c,
                                            const Chunk& lo, const Chunk& hi, bool biased, const Chunk& b0,
                                            const Chunk& b1, const float* cosines, const float* sines, bool live) {
    constexpr int kItems = kHd / 16, kHalf = kHd / 2;
    f32x8 x0 = unpack(lo), x1 = unpack(hi);
    if (biased) {
        const f32x8 y0 = unpack(b0), y1 = unpack(b1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x0[i] += y0[i];
            x1[i] += y1[i];
        }
    }
    if (kind != 2) {
        const f32x8 cv = *reinterpret_cast<const f32x8*>(cosines + 8 * c);
        const f32x8 sv = *reinterpret_cast<const f32x8*>(sines + 8 * c);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const Pair y = rotate(x0[i], x1[i], cv[i], sv[i]);
            x0[i] = y.lo;
            x1[i] = y.hi;
        }
    }
    if (!live || slot < 0 || slot >= a.n_slots) return;
    const Chunk y0 = pack(x0), y1 = pack(x1);
    if (kind == 0) {
        Chunk* dst = reinterpret_cast<Chunk*>(a.q_out + (row * a.nq + h) * kHd) + c;
        store_chunk_as<kStream>(dst, y0);
        store_chunk_as<kStream>(dst + kItems, y1);
    } else {
        void* store = kind == 1 ? a.k_store : a.v_store;
        const size_t at = ((size_t)slot * a.nkv + h) * kHd + 8 * c;
        store_values<kFmt, kStream>(store, at, y0);
        store_values<kFmt, kStream>(store, at + kHalf, y1);
    }
}
// Head `head` of a row, counted q, k, v: which tensor, and the head in it.
__device__ __forceinline__ int kind_of(AppendArgs a, int head, int& h) {
    const int kind = head < a.nq ? 0 : head < a.nq + a.nkv ? 1 : 2;
    h = kind == 0 ? head : kind == 1 ? head - a.nq : head - a.nq - a.nkv;
    return kind;
}
template <int kHd>
__device__ __forceinline__ const Chunk* item_of(AppendArgs a, size_t row, int kind, int h, int c) {
    return reinterpret_cast<const Chunk*>((kind == 0 ? a.q : kind == 1 ? a.k : a.v) +
                                          (row * (kind == 0 ? a.nq : a.nkv) + h) * kHd) + c;
}
template <int kHd>
__device__ __forceinline__ const Chunk* bias_of(AppendArgs a, int kind, int h, int c) {      // or nullptr
    const h16* bias = kind == 0 ? a.q_bias : kind == 1 ? a.k_bias : a.v_bias;
    return bias ? reinterpret_cast<const Chunk*>(bias + (size_t)h * kHd) + c : nullptr;
}

// One row a workgroup, one item a thread (rows of 128 to 1024 items). Position and slot are asked for before the tensors:
// memory returns in order, so the angles are computed while the tensors fly. They go through the vector path, for
// which a zero that the compiler cannot see through stands in: as the scalar loads it makes of a workgroup's one slot
// and position, 14449 rows take 46.5 us instead of 45.8. (Two rows a workgroup: 45.7 us, and 9.2 instead of 8.6 for 2161
// rows into an E4M3 pool; three rows are slower throughout.)
template <int kHd, int kFmt, bool kStream>
__global__ __launch_bounds__(kAppendThreads) void append_row(AppendArgs a, FreqTable freqs) {
    constexpr int kItems = kHd / 16, kHalf = kHd / 2;
    __shared__ __attribute__((aligned(16))) float cs_cos[kHalf], cs_sin[kHalf];
    const int tid = (int)threadIdx.x;
    const size_t row = blockIdx.x;
    const int per_row = (a.nq + 2 * a.nkv) * kItems, item = min(tid, per_row - 1);
    int zero = 0;
    asm volatile("" : "+v"(zero));
    int my_pos = a.positions[row + zero];
    float my_freq = freqs.f[tid % kHalf];
    const int64_t slot = a.slots[row + zero];
    const int c = item % kItems;
    int h;
    const int kind = kind_of(a, item / kItems, h);
    const Chunk* p = item_of<kHd>(a, row, kind, h, c);
    const Chunk lo = load_chunk(p), hi = load_chunk(p + kItems);
    const Chunk* bp = bias_of<kHd>(a, kind, h, c);
    Chunk b0 = {}, b1 = {};
    if (bp) {
        b0 = load_chunk(bp);
        b1 = load_chunk(bp + kItems);
    }
    asm volatile("" : "+v"(my_pos), "+v"(my_freq));
    if (tid < kHalf) {
        float s, cc;
        sincosf((float)my_pos * my_freq, &s, &cc);
        cs_cos[tid] = cc;
        cs_sin[tid] = s;
    }
    __syncthreads();
    finish_item<kHd, kFmt, kStream>(a, row, slot, kind, h, c, lo, hi, bp != nullptr, b0, b1, cs_cos, cs_sin, tid < per_row);
}

// Several rows a workgroup where they are short, several rounds of items where they are very long.
template <int kHd, int kFmt>
__global__ __launch_bounds__(kAppendThreads) void append_rows(AppendArgs a, FreqTable freqs, int rows_per_wg) {
    constexpr int kItems = kHd / 16, kHalf = kHd / 2;
    __shared__ __attribute__((aligned(16))) float cs_cos[kAppendRows * kHalf], cs_sin[kAppendRows * kHalf];
    const int tid = (int)threadIdx.x;
    const int row0 = (int)blockIdx.x * rows_per_wg, rows = min(rows_per_wg, a.rows - row0);
    const int per_row = (a.nq + 2 * a.nkv) * kItems, items = rows * per_row;
    for (int i = tid; i < rows * kHalf; i += (int)blockDim.x) {
        float s, cc;
        sincosf((float)a.positions[row0 + i / kHalf] * freqs.f[i % kHalf], &s, &cc);
        cs_cos[i] = cc;
        cs_sin[i] = s;
    }
    __syncthreads();
    for (int item = tid; item < items; item += (int)blockDim.x) {
        const int r = item / per_row, in_row = item - r * per_row, c = in_row % kItems;
        const size_t row = (size_t)(row0 + r);
        int h;
        const int kind = kind_of(a, in_row / kItems, h);
        const int64_t slot = a.slots[row];
        const Chunk* p = item_of<kHd>(a, row, kind, h, c);
        const Chunk lo = load_chunk(p), hi = load_chunk(p + kItems);
        const Chunk* bp = bias_of<kHd>(a, kind, h, c);
        Chunk b0 = {}, b1 = {};
        if (bp) {
            b0 = load_chunk(bp);
            b1 = load_chunk(bp + kItems);
        }
        finish_item<kHd, kFmt, false>(a, row, slot, kind, h, c, lo, hi, bp != nullptr, b0, b1, cs_cos + r * kHalf,
                                      cs_sin + r * kHalf, true);
    }
}

// Any even head_dim <= 256, any alignment, FP16 pools: a workgroup per row, 2-byte accesses.
__global__ __launch_bounds__(kBlock) void append_generic(AppendArgs a, FreqTable freqs) {
    __shared__ float cs_cos[kMaxPairs];
    __shared__ float cs_sin[kMaxPairs];
    const int half = a.head_dim / 2;
    const size_t row = blockIdx.x;
    const int64_t slot = a.slots[row];
    if (slot < 0 || slot >= a.n_slots) return;
    const int pos = a.positions[row];
    for (int i = (int)threadIdx.x; i < half; i += kBlock) {
        float s, c;
        sincosf((float)pos * freqs.f[i], &s, &c);
        cs_cos[i] = c;
        cs_sin[i] = s;
    }
    __syncthreads();
    const int tasks = (a.nq + 2 * a.nkv) * half;
    for (int t = (int)threadIdx.x; t < tasks; t += kBlock) {
        const int head = t / half, i = t - head * half;
        const int kind = head < a.nq ? 0 : head < a.nq + a.nkv ? 1 : 2;
        const int h = kind == 0 ? head : kind == 1 ? head - a.nq : head - a.nq - a.nkv;
        const size_t in = (row * (size_t)(kind == 0 ? a.nq : a.nkv) + (size_t)h) * (size_t)a.head_dim;
        const h16* src = (kind == 0 ? a.q : kind == 1 ? a.k : a.v) + in;
        const h16* bias = kind == 0 ? a.q_bias : kind == 1 ? a.k_bias : a.v_bias;
        float x0 = (float)src[i], x1 = (float)src[i + half];
        if (bias) {
            x0 += (float)bias[(size_t)h * a.head_dim + i];
            x1 += (float)bias[(size_t)h * a.head_dim + i + half];
        }
        if (kind != 2) {
            const Pair r = rotate(x0, x1, cs_cos[i], cs_sin[i]);
            x0 = r.lo;
            x1 = r.hi;
        }
        h16* dst = kind == 0 ? a.q_out + in
                             : static_cast<h16*>(kind == 1 ? a.k_store : a.v_store) +
                                   ((size_t)slot * a.nkv + (size_t)h) * (size_t)a.head_dim;
        dst[i] = to_half(x0);
        dst[i + half] = to_half(x1);
    }
}

inline bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

}  // namespace
}  // namespace vv

extern "C" {

vv_status_t vv_kv_page_plan_dev(const int* new_lens, const int* cache_lens, int n_seqs, int* page_tables,
                                int max_pages, const int* free_pages, const int* n_free, int* lens_out,
                                int* row_starts, int* positions, int64_t* slots, int max_rows, int* n_free_out,
                                int* counts, void* stream) {
    if (n_seqs <= 0) return VV_OK;
    if (!new_lens || !cache_lens || !page_tables || !free_pages || !n_free || !lens_out || !row_starts || !counts)
        return VV_ERR_NULL_PTR;
    if (max_pages <= 0 || max_rows < 0) return VV_ERR_INVALID_ARG;
    // A saturated row count is past every row then; the loop over sequences, and a position, stay within 32 bits.
    if (max_rows > (1 << 30) || n_seqs > (1 << 30) || (int64_t)max_pages * vv::kPage > INT32_MAX) return VV_ERR_UNSUPPORTED;
    if (max_rows > 0 && (!positions || !slots)) return VV_ERR_NULL_PTR;
    if (lens_out == new_lens || counts == n_free || counts == n_free_out) return VV_ERR_INVALID_ARG;
    vv::PlanArgs a = {new_lens, cache_lens, page_tables, free_pages, n_free, lens_out, row_starts, positions, slots,
                      n_free_out, counts, n_seqs, max_pages, max_rows, max_rows};
    const int threads = n_seqs <= 64 && max_rows <= 64 ? 64 : n_seqs <= 256 ? 256 : vv::kPlanThreads;
    // In place the lengths (or the free count) that a workgroup still has to read are what another writes: one
    // workgroup then, which reads before it writes.
    const bool in_place = lens_out == cache_lens || n_free_out == n_free;
    if (!in_place && max_rows > threads) a.rows_per_wg = threads;
    const unsigned wgs = a.rows_per_wg > 0 ? (unsigned)((max_rows - 1) / a.rows_per_wg + 1) : 1u;
    vv::page_plan<<<dim3(wgs), (unsigned)threads, 0, vv::as_stream(stream)>>>(a);
    return vv::launch_status();
}

vv_status_t vv_rope_kv_append_dev(const void* q, const void* k, const void* v, const void* q_bias,
                                  const void* k_bias, const void* v_bias, const int* positions,
                                  const int64_t* slots, void* q_out, void* k_store, void* v_store, int n_rows,
                                  int n_q_heads, int n_kv_heads, int head_dim, int n_pages, int kv_format,
                                  float theta, void* stream) {
    if (n_rows <= 0) return VV_OK;
    if (!q || !k || !v || !positions || !slots || !q_out || !k_store || !v_store) return VV_ERR_NULL_PTR;
    if (n_q_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 || n_pages <= 0) return VV_ERR_INVALID_ARG;
    if ((head_dim & 1) || head_dim > 2 * vv::kMaxPairs) return VV_ERR_UNSUPPORTED;
    const bool fp8 = kv_format == vv::kFmtE4M3 || kv_format == vv::kFmtE5M2;
    if (kv_format != vv::kFmtFp16 && !(fp8 && head_dim == 128)) return VV_ERR_UNSUPPORTED;
    if ((int64_t)n_q_heads + 2 * (int64_t)n_kv_heads > (1 << 20)) return VV_ERR_UNSUPPORTED;
    const vv::AppendArgs a = {static_cast<const vv::h16*>(q), static_cast<const vv::h16*>(k),
                              static_cast<const vv::h16*>(v), static_cast<const vv::h16*>(q_bias),
                              static_cast<const vv::h16*>(k_bias), static_cast<const vv::h16*>(v_bias), positions,
                              slots, static_cast<vv::h16*>(q_out), k_store, v_store,
                              (int64_t)n_pages * vv::kPage, n_rows, n_q_heads, n_kv_heads, head_dim};
    const vv::FreqTable& freqs = vv::host_freqs(theta, head_dim);
    hipStream_t st = vv::as_stream(stream);
    const bool chunks = vv::aligned16(q) && vv::aligned16(k) && vv::aligned16(v) && vv::aligned16(q_out) &&
                        vv::aligned16(q_bias) && vv::aligned16(k_bias) && vv::aligned16(v_bias) &&
                        (fp8 ? vv::aligned8(k_store) && vv::aligned8(v_store)
                             : vv::aligned16(k_store) && vv::aligned16(v_store));
    if (fp8 && !chunks) return VV_ERR_UNSUPPORTED;
    // A launch holds less than 2^32 threads.
    auto too_many = [](size_t wgs, size_t threads) { return wgs > UINT32_MAX / threads; };
    if (chunks && (head_dim == 128 || head_dim == 64)) {
        const int64_t per_row = (int64_t)(n_q_heads + 2 * n_kv_heads) * (head_dim / 16);
        const bool one = per_row >= 128 && per_row <= vv::kAppendThreads;
        int rows = per_row >= 128 ? 1 : (int)(256 / per_row);
        if (rows > vv::kAppendRows) rows = vv::kAppendRows;
        if (rows > n_rows) rows = n_rows;
        const int64_t want = (rows * per_row + vv::kWave - 1) / vv::kWave * vv::kWave;
        const unsigned threads = (unsigned)(want < vv::kAppendThreads ? want : vv::kAppendThreads);
        const dim3 grid((unsigned)((n_rows - 1) / rows + 1));
        if (too_many(grid.x, threads)) return VV_ERR_UNSUPPORTED;
        const bool stream = vv::use_streaming(2u * (size_t)n_rows * (size_t)per_row * 32u);
#define VV_APPEND(H, F)                                                                        \
    do {                                                                                       \
        if (one && stream) vv::append_row<H, vv::F, true><<<grid, threads, 0, st>>>(a, freqs); \
        else if (one)      vv::append_row<H, vv::F, false><<<grid, threads, 0, st>>>(a, freqs); \
        else               vv::append_rows<H, vv::F><<<grid, threads, 0, st>>>(a, freqs, rows); \
    } while (0)
        if (head_dim == 64)                       VV_APPEND(64, kFmtFp16);
        else if (!fp8)                            VV_APPEND(128, kFmtFp16);
        else if (kv_format == vv::kFmtE4M3)       VV_APPEND(128, kFmtE4M3);
        else                                      VV_APPEND(128, kFmtE5M2);
#undef VV_APPEND
    } else {
        if (too_many((size_t)n_rows, vv::kBlock)) return VV_ERR_UNSUPPORTED;
        vv::append_generic<<<dim3((unsigned)n_rows), vv::kBlock, 0, st>>>(a, freqs);
    }
    return vv::launch_status();
}

}  // extern "C"
