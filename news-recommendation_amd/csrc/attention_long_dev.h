// device pieces shared by the forward and backward kernels of attention_long*.hip
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
    int causal, additive, drop;
    float scale, fill, keep;                    // keep = 1 / (1 - p)
    uint32_t thr, site;
    uint64_t seed;
    // forward
    void* out; AttnStrides so;
    float *row_max, *row_sum;
    // backward
    const void* dout; AttnStrides sdo;
    float* delta; AttnStrides sd;
    void *dq, *dk, *dv; AttnStrides sdq, sdk, sdv;
    // split of the long axis
    float* part; float* part_ml;
    int nblk_r;                                 // row (dKV: key) blocks of one key head
    int splits, per_split;
};

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float NEVER = -1e30f;                 // running maximum before the first key: finite, so exp2(-inf - NEVER) = 0 and no inf - inf

// neighbouring workgroups go to different XCDs; this order gives each XCD a contiguous run of the logical ones, so that blocks
// which read the same key head share an L2
__device__ __forceinline__ uint32_t xcd_order(uint32_t b, uint32_t n) {
    const uint32_t x = b & 7, q = n >> 3, rem = n & 7;
    return x * q + (x < rem ? x : rem) + (b >> 3);
}
// the causal rows' work grows with the row: heavy and light blocks alternate within a head
__device__ __forceinline__ int heavy_light(int i, int n) { return (i & 1) ? (i >> 1) : n - 1 - (i >> 1); }

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

// A [ROWS x DHP] tile on its way from global memory into LDS, 16 bytes per piece: `load` only issues the loads, `store` waits.
// row_ptr(row) gives the row's address, or NULL for a row that has to read as zero.
template <class T, int DHP, int ROWS, bool VEC>
struct Stage {
    static constexpr int E = Ty<T>::E, PITCH = DHP + Ty<T>::PAD, PER_ROW = DHP / E, NCH = ROWS * PER_ROW / 256;
    static_assert(ROWS * PER_ROW % 256 == 0, "whole pieces per thread");
    u32x4 r[NCH];
    template <class F> __device__ __forceinline__ void load(int tid, int dh, F row_ptr) {
#pragma unroll
        for (int u = 0; u < NCH; ++u) {
            const int c = tid + 256 * u, row = c / PER_ROW, col = (c % PER_ROW) * E;
            const T* p = row_ptr(row);
            r[u] = load16<T, VEC>(p + col, p ? dh - col : 0);
        }
    }
    template <class F> __device__ __forceinline__ void store(int tid, T* lds, F keep) {
#pragma unroll
        for (int u = 0; u < NCH; ++u) {
            const int c = tid + 256 * u, row = c / PER_ROW, col = (c % PER_ROW) * E;
            *reinterpret_cast<u32x4*>(lds + row * PITCH + col) = keep(row) ? r[u] : u32x4{0, 0, 0, 0};
        }
    }
};

// presence bits of the WORDS * 64 keys from j on.  load() issues, bits() waits; every wave holds all of them
template <int WORDS>
struct KeyBits {
    int64_t m[WORDS];
    __device__ __forceinline__ void load(const int64_t* mask, int j, int end, int lane) {
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
            const int key = j + 64 * w + lane;
            m[w] = mask ? (key < end ? mask[key] : 0) : (key < end);
        }
    }
    __device__ __forceinline__ uint64_t bits(int w) const { return __ballot(m[w] != 0); }
};

// the end of the keys a block has to read: `end`, less whole runs of 256 absent keys at the end of [begin, end)
__device__ __forceinline__ int present_end(const int64_t* mask, int begin, int end, int tid) {
    while (end > begin) {
        const int j = end - 256 + tid;
        const int there = j >= begin && mask[j] != 0;
        if (__syncthreads_or(there)) break;
        end -= 256;
    }
    return end > begin ? end : begin;
}

// [sub] x 16 scores of this lane's row -> the same with what the row must not see taken out.  key0: the key of register 0's row 0
__device__ __forceinline__ void hide(f32x16& x, uint32_t bits, int key0, int lim, int h) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int t = tile_row(r, h);
        if (!((bits >> t) & 1) || key0 + t > lim) x[r] = -INFINITY;
    }
}

// host side
Args make_args(const AttnProblem& p);
bool aligned16(const void* ptr, const AttnStrides& st, int dh, size_t elem);
bool all_aligned(const AttnProblem& p);
struct Split { int splits, per; };
Split split_axis(int64_t blocks, int length, int unit);

}  // namespace al
}  // namespace nr
