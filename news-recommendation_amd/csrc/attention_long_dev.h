// device pieces shared by the forward and backward kernels of attention of any length (attention_long_fwd.h, attention_long_bwd.h)
#pragma once
#include "attention_long.h"
#include "mma.h"

namespace nr {
namespace al {

using namespace mma;

// kernel arguments (by value)
struct Args {
    const void *q, *k, *v;
    const int64_t* mask;
    AttnStrides sq, sk, sv;
    int64_t N;
    int Sq, Sk, H, G, rep, dh, dhs;             // rep = H / G; dhs = dh rounded up to 4 (row length of the partial results)
    int R;                                      // rep * Sq: the rows of one key head (query head major)
    int causal, additive;
    float scale, fill, keep;                    // keep = 1 / (1 - p)
    uint32_t thr, site;
    uint64_t seed;
    // forward
    void* out; AttnStrides so;
    float *row_max, *row_sum;
    // backward
    const void* dout; AttnStrides sdo;
    float* delta; AttnStrides sd;
    int keep_delta;                             // the dQ pass runs first and writes delta
    void *dq, *dk, *dv; AttnStrides sdq, sdk, sdv;
    // split of the long axis
    float* part; float* part_ml;
    int nblk;                                   // row (dKV: key) blocks of one key head
    int head_blocks;                            // > 0: row blocks of one query head, none of which reaches into the next head
    int splits, per_split;
};

// what tensors of type T are multiplied as: fp32 in three parts, except with WK = 4 (few rows: bound by memory and latency)
template <class T, int WK> struct MulType { typedef T M; };
template <> struct MulType<float, 1> { typedef Split3 M; };

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NEVER = -3.402823466e38f;       // running maximum before the first key: finite, so exp2(-inf - NEVER) = 0 and no inf - inf

// Neighbouring workgroups go to different XCDs, each with its own L2.  Key heads are dealt to the XCDs, so that the workgroups of one
// head share an L2 and sequences of different lengths still spread over the chip; what is left of a multiple of 8 heads is spread
// block by block.  (Contiguous runs of blocks per XCD, which this replaced, left XCDs idle whenever neighbouring sequences were
// short: 32 x 512 with lengths 128 .. 512 took as long as 32 x 512 without padding.)
struct Slot { int head, w; };                   // key head (n * G + g), block of that head
__device__ __forceinline__ Slot deal(uint32_t b, uint32_t heads, uint32_t per_head) {
    const uint32_t full = heads & ~7u;
    if (b < full * per_head) {
        const uint32_t slot = b >> 3, q = slot / per_head;
        return Slot{(int)(q * 8 + (b & 7)), (int)(slot - q * per_head)};
    }
    b -= full * per_head;
    const uint32_t left = heads - full, w = b / left;
    return Slot{(int)(full + b - w * left), (int)w};
}
// rows [r0, rend) of row block w: with causal order the blocks with most keys come first, one query head per block
struct Rows { int r0, rend; };
__device__ __forceinline__ Rows row_block(const Args& a, int w, int rows) {
    if (!a.head_blocks) return Rows{w * rows, a.R};
    const int p = w / a.rep, hh = w - p * a.rep;
    return Rows{hh * a.Sq + (a.head_blocks - 1 - p) * rows, (hh + 1) * a.Sq};
}

// keep bits of the probabilities (row_linear, j) .. (row_linear, j + 3): element index row_linear * Sk + j of the library's stream
__device__ __forceinline__ uint32_t keep4(const Args& a, uint64_t idx) {
    const Philox4 x = philox4x32_10(a.seed, idx >> 2, a.site);
    const int o = (int)(idx & 3);
    uint32_t w[7] = {x.x, x.y, x.z, x.w, 0, 0, 0};
    if (o) {
        const Philox4 y = philox4x32_10(a.seed, (idx >> 2) + 1, a.site);
        w[4] = y.x; w[5] = y.y; w[6] = y.z;
    }
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t v = o == 0 ? w[e] : (o == 1 ? w[e + 1] : (o == 2 ? w[e + 2] : w[e + 3]));
        m |= (v >= a.thr ? 1u : 0u) << e;
    }
    return m;
}

// Rows [0, rows) of a [ROWS x DHP] tile on their way from global memory into LDS, 16 bytes per piece: `load` only issues the loads,
// `store` waits.  Rows past `rows` and columns past dh read as zero, except that rows which share memory (a row stride below dh) may
// go on with what is left of it: finite where the rows are, and no memory of others.  VEC: buffer loads whose bounds check does that,
// with one 32-bit offset per thread (the host checks that a tile's offsets fit); otherwise element by element.
template <class T, int DHP, int ROWS, bool VEC, int NT = 256>
struct Stage {
    static constexpr int E = Ty<T>::E, PER_ROW = DHP / E, NCH = ROWS * PER_ROW / NT, STEP = NT / PER_ROW;
    static_assert(ROWS * PER_ROW % NT == 0 && NT % PER_ROW == 0, "whole pieces per thread, whole rows per pass");
    u32x4 r[NCH];
    int row, col, width, pitch;                 // this thread's first piece; columns, and elements from row to row (VEC)
    uint32_t voff;
    int64_t stride;
    __device__ __forceinline__ void setup(int tid, int64_t row_stride, int columns) {
        row = tid / PER_ROW;
        col = (tid % PER_ROW) * E;
        width = columns;
        stride = row_stride;
        pitch = (int)row_stride;
        voff = col < width ? (uint32_t)(row * pitch + col) * (uint32_t)sizeof(T) : 0x80000000u;
    }
    __device__ __forceinline__ void load(const T* base, int rows) {
        if (VEC) {
            const int n = rows < ROWS ? rows : ROWS;                             // (so the tile's extent fits 32 bits)
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<T*>(base), 0, n > 0 ? ((n - 1) * pitch + width) * (int)sizeof(T) : 0, 0x00020000);
#pragma unroll
            for (int u = 0; u < NCH; ++u) r[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(voff + u * (uint32_t)(STEP * pitch * (int)sizeof(T))), 0, 0);
        } else {
#pragma unroll
            for (int u = 0; u < NCH; ++u)
                r[u] = load16<T, false>(base + (row + STEP * u) * stride + col, row + STEP * u < rows ? width - col : 0);
        }
    }
    template <class L> __device__ __forceinline__ void store(char* lds) const {              // L: the tile's layout (mma.h)
#pragma unroll
        for (int u = 0; u < NCH; ++u) L::put(lds, row + STEP * u, col, r[u]);
    }
    template <class L, class F> __device__ __forceinline__ void store_if(char* lds, F keep) const {
#pragma unroll
        for (int u = 0; u < NCH; ++u) L::put(lds, row + STEP * u, col, keep(row + STEP * u) ? r[u] : u32x4{0, 0, 0, 0});
    }
};

// Which keys are there, a bit each, for up to SPAN keys from `from` on: read once, kept in LDS.  Without a mask the bits follow from
// the end alone.
constexpr int SPAN = 8192;
struct KeyBits {
    uint64_t* words;                            // [SPAN / 64] in LDS
    bool masked;
    int from, end;                              // keys [from, end)
    // all threads; returns the end of the last key that is there (>= from)
    __device__ __forceinline__ int fill(const int64_t* mask, int lane, int wave) {
        const int n = (end - from + 63) >> 6;
#pragma unroll 4
        for (int x = wave; x < n; x += 4) {
            const int key = from + 64 * x + lane;
            const uint64_t b = __ballot(key < end && mask[key] != 0);
            if (lane == 0) words[x] = b;
        }
        __syncthreads();
        const uint64_t lo = __ballot(lane < n && words[lane] != 0), hi = __ballot(64 + lane < n && words[64 + lane] != 0);
        if (!(lo | hi)) return from;
        const int top = hi ? 127 - __builtin_clzll(hi) : 63 - __builtin_clzll(lo);
        return from + 64 * top + 64 - __builtin_clzll(words[top]);
    }
    __device__ __forceinline__ uint64_t range(int j) const {
        const int left = end - j;
        return left >= 64 ? ~0ull : (left > 0 ? (1ull << left) - 1 : 0ull);
    }
    // 64 keys from j (a multiple of 32 past `from`) on; wave-uniform
    __device__ __forceinline__ uint64_t at(int j) const {
        if (!masked) return range(j);
        if (j >= end) return 0;
        const int x = (j - from) >> 6;
        const uint64_t w = words[x];
        const uint64_t u = (uint64_t)__builtin_amdgcn_readfirstlane((int)(w >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)w);
        return ((j - from) & 32) ? u >> 32 : u;
    }
};

// scores of this lane's row, 16 keys of 32 from key0 on: what the row must not see becomes -inf.  The keys that are not there are the
// same for every row: one wave-wide select per register; the causal end is the lane's own.
__device__ __forceinline__ void hide(f32x16& x, uint32_t bits, int key0, int lim, int lim_min, int h) {
    if (bits != ~0u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int t = tile_row(r, 0);
            const uint64_t on = ((bits >> t) & 1 ? 0xffffffffull : 0) | ((bits >> (t + 4)) & 1 ? 0xffffffffull << 32 : 0);
            x[r] = __builtin_amdgcn_inverse_ballot_w64(on) ? x[r] : -INFINITY;
        }
    if (key0 + 31 > lim_min) {
        const int last = lim - key0 - 4 * h;
#pragma unroll
        for (int r = 0; r < 16; ++r) x[r] = tile_row(r, 0) <= last ? x[r] : -INFINITY;
    }
}

// host side
// 16-byte loads and stores: the address and every stride a multiple of 16 bytes; `tile` rows of it within a 32-bit offset
inline bool aligned16(const void* ptr, const AttnStrides& st, int dh, size_t elem, int tile) {
    const int64_t e = 16 / (int64_t)elem;
    return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && dh % e == 0 && st.n % e == 0 && st.s % e == 0 && st.h % e == 0 &&
           st.s >= 0 && st.s < ((int64_t)1 << 31) / (tile * (int64_t)elem);
}
Args make_args(const AttnProblem& p);
template <class T> int run_fwd(const Args& a, bool vec, bool drop, int wk, unsigned grid, hipStream_t s);
struct Split { int splits, per; };
struct BwdPlan { int wk, nblk_q, nblk_k, head_blocks; Split q, kv; size_t ws; };
template <class T> int run_bwd(Args a, const BwdPlan& f, bool vec, bool drop, bool room, hipStream_t s);

}  // namespace al
}  // namespace nr
