// Linear attention with a decay for each head, chunked.
//
//   S_t = w S_{t-1} + k_t v_t^T,  o_t = scale * q_t S_t   (w = e^{log_decay[h]}, S_t [dk,dv])
//
// A chunk of 32 tokens that starts from state S gives, with i, j positions in the chunk and m its token count,
//   o_i = scale * ( sum_{j <= i} w^{i-j} (q_i . k_j) v_j  +  w^{i+1} q_i S ),     S' = w^m S + sum_i w^{m-1-i} k_i v_i^T
// so everything is a matrix product; the powers are of exponents >= 0 (no overflow however fast a head forgets).
//
// The backward is the same form three times over: with g = dO,
//   dq_t = scale * sum_{s <= t} w^{t-s} (g_t . v_s) k_s           = the forward of (g, v, k), starting from S_0^T
//   dk_s = sum_{t >= s} w^{t-s} scale (v_s . g_t) q_t             = from the other end, (v, g, q), starting from dS_last^T
//   dv_s = sum_{t >= s} w^{t-s} scale (k_s . q_t) g_t             = from the other end, (k, q, g), starting from dS_last; it ends in dS_0
// From the other end (rev) the carried state R already holds the step to the next token: o_i = sum_{j >= i} w^{j-i} (..) + w^{m-1-i} x_i R,
// R' = w^m R + sum_i w^{i+1} y_i z_i^T.  One kernel computes o = form(x, y, z) for all of them; the three of a backward are one launch,
// neighbours on one XCD, so that what they read twice comes from its L2.
//
// Work split.  A wave owns 32 columns of z / o and of the state, which stays in its registers in fp32 (rows a, column b: a D tile,
// mma.h) for the whole walk; a workgroup has one wave per 32 columns (bf16 heads of up to 64: two, lin_pair_kernel).  Registers feed both products of the state: as D tiles they
// are the A operand of o^T += S^T x^T without a transpose, and the z fragments are the A operand of o^T += z^T A^T and the B
// operand of S += y^T z.  When heads * sequences do not fill the chip the tokens are also cut into segments: every segment's own
// sum first (lin_state), a scan over them (lin_scan), then the walk with the right starting states.
//
// Rounding (bf16): the decayed scores, and the state where a query meets it, are rounded to bf16 as operands of a product (half a
// step each, against an output of the same type); what goes INTO the state is not (Weighed), and every sum, and the state from chunk
// to chunk, is fp32.
//
// Measured (MI355X, bf16, heads of 64).  What bounds it is the chain through the state: the tiles of a sequence follow one another, and
// one wave for everything took about 7300 cycles per 64 tokens (scores and output 1180 and state 1330 per chunk, stores 400, LDS 510,
// loads 430), which the pairs of waves divide.  32 sequences up to 1000 tokens, 12 heads: forward 60 us (73 with one wave), backward 100
// (111).  2 x 16384 tokens, 12 heads, in 32 segments: segment sums 26 us, scan 9 us, output 45 us: 2.5 TB/s in all, 3.8 with the
// second read of k and v.  128 x 1000 tokens, 12 heads: forward 201 us, 3.9 TB/s.  One wave for everything, the same 32 sequences: bf16,
// 128 wide: forward 147 us, backward 320; fp32, 64 wide (on the fp32 matrix instruction): 201 and 265; 128 wide a pass of both 1250.
// lin_pair_kernel at unaligned 64 x 32 widths puts 17 registers per lane into scratch memory, lin_out_kernel at unaligned 128 x 32 in bf16 25.
#include "linear_attention.h"
#include "attention_long_dev.h"
#include <algorithm>

namespace nr {
namespace lin {

using namespace mma;

constexpr int UNIT = 64;                         // segments are multiples of this many tokens
template <class T> constexpr int TILE = sizeof(T) == 2 ? 64 : 32;        // tokens per LDS tile: two chunks of bf16, one of fp32

struct Job {
    const void *x, *y, *z;
    AttnStrides sx, sy, sz, so;
    void* o;
    const float* init; int init_t;               // starting state [da,db] (init_t: stored [db,da]), NULL: zero
    float* last;                                 // final state [da,db], NULL: not wanted
    float* seg;                                  // [N*H][G][da*db]: segment sums, then starting states
    int da, db, rev;
    float amul, imul, umul;                      // factors of the scores, of the state's product, of what is added to the state
};
struct Args {
    Job job[3];
    int jobs, G, per;                            // segments of `per` tokens (a multiple of UNIT)
    int64_t N;
    int S, H;
    const float* log_decay;
    const int64_t* lens;
};

__device__ __forceinline__ float power(float a2, int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f(a2 * (float)n); }
__device__ __forceinline__ int length_of(const Args& a, int64_t n) {
    if (!a.lens) return a.S;
    const int64_t l = a.lens[n];
    return (int)(l < 0 ? 0 : (l > a.S ? a.S : l));
}
// 8 elements of a row in "tile" order: p points at column 16 * kstep + 4 * h
__device__ __forceinline__ bf16x8 spread_frag(const __bf16* p) {
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(p), b = *reinterpret_cast<const bf16x4*>(p + 8);
    return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
__device__ __forceinline__ f32x8 spread_frag(const float* p) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 8);
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
// what a chunk adds to the state: S += y^T (w z), k-step kb of it.  bf16: w z goes in as a sum of bf16 numbers, three of them (its
// fp32 value to the last bit but one) where the state is a result of the call, in fp32, or where segments start from it; two where
// it only meets the queries of a bf16 output.  (The final state of 1000 tokens: off by 4e-7 of its norm with three, as in fp32
// throughout; 2.5e-6 with two, 2.8e-3 with one.)
template <class T, int PIECES> struct Weighed;
template <int PIECES> struct Weighed<float, PIECES> {
    f32x8 v;
    __device__ __forceinline__ Weighed(const f32x8& z, const float* w, int h) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(w + 4 * h), b = *reinterpret_cast<const f32x4*>(w + 8 + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = z[e] * a[e]; v[4 + e] = z[4 + e] * b[e]; }
    }
    __device__ __forceinline__ f32x16 add(const f32x8& y, const f32x16& s) const { return mul(y, v, s); }
};
template <int PIECES> struct Weighed<__bf16, PIECES> {
    u32x4 v[PIECES];
    __device__ __forceinline__ Weighed(const bf16x8& z, const float* w, int h) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(w + 4 * h), b = *reinterpret_cast<const f32x4*>(w + 8 + 4 * h);
        const u32x4 u = __builtin_bit_cast(u32x4, z);
#pragma unroll
        for (int e = 0; e < 4; ++e) {            // two elements at a time
            float x = __uint_as_float(u[e] << 16) * (e < 2 ? a[2 * e] : b[2 * e - 4]);
            float y = __uint_as_float(u[e] & 0xffff0000u) * (e < 2 ? a[2 * e + 1] : b[2 * e - 3]);
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                v[i][e] = pack2(x, y);
                x -= __uint_as_float(v[i][e] << 16);
                y -= __uint_as_float(v[i][e] & 0xffff0000u);
            }
        }
    }
    __device__ __forceinline__ f32x16 add(const bf16x8& y, f32x16 s) const {
#pragma unroll
        for (int i = PIECES - 1; i >= 0; --i) s = mul(y, __builtin_bit_cast(bf16x8, v[i]), s);
        return s;
    }
};

// where a workgroup stands: job, head, segment
struct Place {
    int job, seg, h, s0, s1, send;
    int64_t n, nh;
    float a2;
    __device__ __forceinline__ Place(const Args& a) {
        const al::Slot slot = al::deal(blockIdx.x, (uint32_t)(a.N * a.H), a.G * a.jobs);
        nh = slot.head;
        seg = slot.w / a.jobs;
        job = slot.w - seg * a.jobs;
        n = nh / a.H;
        h = (int)(nh - n * a.H);
        a2 = a.log_decay[h] * al::LOG2E;
        s0 = seg * a.per;
        send = min(a.S, s0 + a.per);
        s1 = max(s0, min(length_of(a, n), send));
    }
};

// the weights of what m of a chunk's 32 tokens add to the state, times umul: w^{m-1-i}, from the other end w^{i+1}; zero behind m
__device__ __forceinline__ float add_weight(float a2, int i, int m, int rev, float umul) {
    return i < m ? umul * power(a2, rev ? i + 1 : m - 1 - i) : 0.f;
}

// the tiles of C tokens that a workgroup walks, the next one on its way from memory while one is worked on
template <class T, int DA, int DB, bool VEC, bool OUT, int NT = 2 * DB> struct Walk {
    static constexpr int PA = DA + Ty<T>::PAD, PB = DB + Ty<T>::PAD, C = TILE<T>;
    static constexpr size_t LDS = ((OUT ? 2 : 1) * PA + PB) * C * sizeof(T) + C * 4 + (OUT ? 64 * 4 : 0);
    typedef Lds<T, C, DA> LA;
    typedef Lds<T, C, DB> LB;
    struct Set {
        al::Stage<T, DA, C, VEC, NT> x, y;
        al::Stage<T, DB, C, VEC, NT> z;
    };
    const Place& at;
    const T *xp = nullptr, *yp, *zp;             // the next tile
    int64_t xstep = 0, ystep, zstep;
    int rev;
    float umul;
    T *Xs, *Ys, *Zs;
    float* wu;
    int had = -1, nc;
    __device__ __forceinline__ Walk(const Place& at, const Job& J, char* smem) : at(at) {
        nc = (at.s1 - at.s0 + C - 1) / C;
        rev = J.rev; umul = J.umul;
        const int64_t first = at.s0 + C * (rev ? nc - 1 : 0), dir = rev ? -C : C;
        if (OUT) { xp = static_cast<const T*>(J.x) + at.n * J.sx.n + at.h * J.sx.h + first * J.sx.s; xstep = dir * J.sx.s; }
        yp = static_cast<const T*>(J.y) + at.n * J.sy.n + at.h * J.sy.h + first * J.sy.s; ystep = dir * J.sy.s;
        zp = static_cast<const T*>(J.z) + at.n * J.sz.n + at.h * J.sz.h + first * J.sz.s; zstep = dir * J.sz.s;
        Ys = reinterpret_cast<T*>(smem);
        Zs = Ys + C * PA;
        Xs = Zs + C * PB;
        wu = reinterpret_cast<float*>(Xs + (OUT ? C * PA : 0));
    }
    __device__ __forceinline__ void setup(Set& s, const Job& J, int tid) const {
        if (OUT) s.x.setup(tid, J.sx.s, J.da);
        s.y.setup(tid, J.sy.s, J.da);
        s.z.setup(tid, J.sz.s, J.db);
    }
    __device__ __forceinline__ int tile(int t) const { return rev ? nc - 1 - t : t; }
    __device__ __forceinline__ int tokens(int t) const { return at.s1 - at.s0 - C * tile(t); }      // from the tile's start on
    __device__ __forceinline__ void fetch(Set& s, int t) {                       // (past the last tile: zeros, no memory is read)
        const int rows = t < nc ? tokens(t) : 0;
        if (OUT) s.x.load(xp, rows);
        s.y.load(yp, rows);
        s.z.load(zp, rows);
        xp += xstep; yp += ystep; zp += zstep;
    }
    // tile t into LDS; returns its token count
    __device__ __forceinline__ int put(const Set& s, int t, int tid) {
        const int m = min(C, tokens(t));
        __syncthreads();
        if (OUT) s.x.template store<LA>(reinterpret_cast<char*>(Xs));
        s.y.template store<LA>(reinterpret_cast<char*>(Ys));
        s.z.template store<LB>(reinterpret_cast<char*>(Zs));
        if (m != had && tid < C) wu[tid] = add_weight(at.a2, tid & 31, min(32, max(0, m - (tid & 32))), rev, umul);
        had = m;
        __syncthreads();
        return m;
    }
};
// S = w^m S + sum over the m tokens of half `it` of the tile; zf: the half's z columns of this wave
template <class T, int PA, int AT, int PIECES>
__device__ __forceinline__ void absorb(f32x16 (&S)[AT], const T* Ys, const float* wu, const typename Ty<T>::Frag (&zf)[2], float all, int it, int lane) {
#pragma unroll
    for (int x = 0; x < AT; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[x][r] *= all;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        const Weighed<T, PIECES> zw(zf[kb], wu + 32 * it + 16 * kb, lane >> 5);
#pragma unroll
        for (int x = 0; x < AT; ++x) S[x] = zw.add(col_frag<PA>(Ys, 32 * it + 16 * kb, 32 * x, lane), S[x]);
    }
}

template <class T, int DA, int DB, bool VEC>
__global__ __launch_bounds__(2 * DB, (DA * sizeof(T) <= 128 ? 3 : (DA * sizeof(T) <= 256 && sizeof(T) == 4 ? 2 : 1))) void lin_state_kernel(const Args a) {
    constexpr int AT = DA / 32;
    typedef Walk<T, DA, DB, VEC, false> W;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Place at(a);
    const Job& J = a.job[at.job];
    W walk(at, J, smem);
    f32x16 S[AT];
#pragma unroll
    for (int t = 0; t < AT; ++t) S[t] = zero16();
    typename W::Set set;
    walk.setup(set, J, tid);
    walk.fetch(set, 0);
    for (int t = 0; t < walk.nc; ++t) {
        const int m = walk.put(set, t, tid);
        walk.fetch(set, t + 1);
#pragma unroll
        for (int u = 0; u < W::C / 32; ++u) {
            const int it = walk.rev ? W::C / 32 - 1 - u : u, mi = min(32, m - 32 * it);
            if (mi <= 0) continue;
            typename Ty<T>::Frag zf[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) zf[kb] = col_frag<W::PB>(walk.Zs, 32 * it + 16 * kb, 32 * w, lane);
            absorb<T, W::PA, AT, 3>(S, walk.Ys, walk.wu, zf, power(at.a2, mi), it, lane);
        }
    }
    float* dst = J.seg + (at.nh * a.G + at.seg) * (int64_t)(J.da * J.db);
    const int b = 32 * w + l31;
    if (b < J.db)
#pragma unroll
        for (int x = 0; x < AT; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * x + tile_row(r, h);
                if (row < J.da) dst[row * J.db + b] = S[x][r];
            }
}

// segment sums -> the states that the segments start from (in place), and the final state
__global__ __launch_bounds__(256) void lin_scan_kernel(const Args a) {
    const Job& J = a.job[blockIdx.y];
    const int64_t E = (int64_t)J.da * J.db, idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= a.N * a.H * E) return;
    const int64_t nh = idx / E, e = idx - nh * E, n = nh / a.H;
    const float a2 = a.log_decay[nh - n * a.H] * al::LOG2E;
    const int len = length_of(a, n);
    float s = 0.f;
    if (J.init) {
        const int64_t row = e / J.db, col = e - row * J.db;
        s = J.init[nh * E + (J.init_t ? col * J.da + row : e)];
    }
    float* p = J.seg + nh * a.G * E + e;
#pragma unroll 8
    for (int t = 0; t < a.G; ++t) {
        const int g = J.rev ? a.G - 1 - t : t;
        const int m = min(max(len - g * a.per, 0), a.per);
        const float add = p[g * E];
        p[g * E] = s;
        s = fmaf(power(a2, m), s, add);
    }
    if (J.last) J.last[nh * E + e] = s;
}

// EXACT: one segment whose final state is wanted
template <class T, int DA, int DB, bool VEC, bool EXACT>
__global__ __launch_bounds__(2 * DB, (DA * sizeof(T) <= 128 ? 3 : (DA * sizeof(T) <= 256 && sizeof(T) == 4 ? 2 : 1))) void lin_out_kernel(const Args a) {
    constexpr int NT = 2 * DB, AT = DA / 32, KA = DA / 16;
    typedef Walk<T, DA, DB, VEC, true> W;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Place at(a);
    const Job& J = a.job[at.job];
    W walk(at, J, smem);
    T* op = static_cast<T*>(J.o) + at.n * J.so.n + at.h * J.so.h;
    const int b = 32 * w + l31;
    const int64_t E = (int64_t)J.da * J.db;
    typename W::Set set;
    walk.setup(set, J, tid);
    walk.fetch(set, 0);

    f32x16 S[AT];
    {
        const float* src = a.G > 1 ? J.seg + (at.nh * a.G + at.seg) * E : (J.init ? J.init + at.nh * E : nullptr);
        const bool turned = a.G == 1 && J.init_t;
#pragma unroll
        for (int x = 0; x < AT; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * x + tile_row(r, h);
                S[x][r] = src && row < J.da && b < J.db ? src[turned ? b * J.da + row : row * J.db + b] : 0.f;
            }
    }
    // decays between 32 tokens, by (row j) - (column i) + 31; zero on the side that the sum leaves out.  (In registers they took the
    // sixteen that a third wave per SIMD needs.)
    float* near = walk.wu + W::C;
    if (tid < 64) {
        const int d = J.rev ? tid - 31 : 31 - tid;
        near[tid] = d >= 0 ? J.amul * power(at.a2, d) : 0.f;
    }
    const float* nearest = near + 31 + 4 * h - l31;
    const float imul = J.imul;
    const int64_t ostep = J.so.s;
    const int db = J.db;
    for (int t = 0; t < walk.nc; ++t) {
        const int t0 = at.s0 + W::C * walk.tile(t), m = walk.put(set, t, tid);
        walk.fetch(set, t + 1);
#pragma unroll 1
        for (int u = 0; u < W::C / 32; ++u) {
            const int it = walk.rev ? W::C / 32 - 1 - u : u, mi = min(32, m - 32 * it);
            if (mi <= 0) continue;
            const T* xr = walk.Xs + (32 * it + l31) * W::PA;
            const T* yr = walk.Ys + (32 * it + l31) * W::PA;
            f32x16 x = zero16(), o = zero16();
#pragma unroll
            for (int k = 0; k < KA; ++k) x = mul(near_frag(yr + 16 * k + 8 * h), near_frag(xr + 16 * k + 8 * h), x);
#pragma unroll
            for (int y = 0; y < AT; ++y)
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2) o = mul(tile_frag<T>(S[y], k2), spread_frag(xr + 32 * y + 16 * k2 + 4 * h), o);
            const float wi = imul * power(at.a2, walk.rev ? max(mi - 1 - l31, 0) : l31 + 1);
#pragma unroll
            for (int r = 0; r < 16; ++r) { o[r] *= wi; x[r] *= nearest[tile_row(r, 0)]; }
            typename Ty<T>::Frag zf[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                zf[kb] = col_frag<W::PB>(walk.Zs, 32 * it + 16 * kb, 32 * w, lane);
                o = mul(zf[kb], tile_frag<T>(x, kb), o);
            }
            if (l31 < mi) {
                T* row = op + (t0 + 32 * it + l31) * ostep;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int col = 32 * w + 8 * q + 4 * h;
                    store4<VEC>(row + col, f32x4{o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]}, db - col);
                }
            }
            absorb<T, W::PA, AT, (EXACT ? 3 : 2)>(S, walk.Ys, walk.wu, zf, power(at.a2, mi), it, lane);
        }
    }
    if (EXACT && J.last && b < J.db)
#pragma unroll
        for (int x = 0; x < AT; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * x + tile_row(r, h);
                if (row < J.da) J.last[at.nh * E + row * J.db + b] = S[x][r];
            }
    // rows behind the sequence's length
    for (int x = tid; x < (at.send - at.s1) * J.db; x += NT) {
        const int row = x / J.db;
        op[(int64_t)(at.s1 + row) * J.so.s + (x - row * J.db)] = (T)0.f;
    }
}

// The same for bf16 heads of up to 64: a pair of waves per 32 columns, one that carries the state through the tiles and hands it on, in
// bf16, as the fragments that the other multiplies while the first goes on.  The chain of a sequence is then the longer of the two
// halves, not their sum.  A tile's second chunk meets the first one's tokens directly (one more block of scores), so that both waves
// work on the same tile and one state per tile is handed over.  (One wave for both, 40 x 12 heads of 1000 x 64: forward 66 us, backward
// 178; pairs 55 and 153.  128 x 12 heads: 223 and 519; 201 and 471.  Wider heads and fp32 would not leave the LDS for it.)
template <int DA, int DB> constexpr bool PAIRED = DA <= 64 && DB <= 64;
template <int DA, int DB, bool VEC, bool EXACT>
__global__ __launch_bounds__(4 * DB, 3) void lin_pair_kernel(const Args a) {
    typedef __bf16 T;
    constexpr int NT = 4 * DB, NB = DB / 32, AT = DA / 32, KA = DA / 16;
    typedef Walk<T, DA, DB, VEC, true, NT> W;
    static_assert(W::C == 64 && W::LDS % 16 == 0, "two chunks per tile");
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool carry = w >= NB;
    const int wb = carry ? w - NB : w, b = 32 * wb + l31;
    const Place at(a);
    const Job& J = a.job[at.job];
    W walk(at, J, smem);
    T* op = static_cast<T*>(J.o) + at.n * J.so.n + at.h * J.so.h;
    const int64_t E = (int64_t)J.da * J.db;
    typename W::Set set;
    walk.setup(set, J, tid);
    walk.fetch(set, 0);
    // decays between tokens of one chunk, by (row j) - (column i) + 31 (zero on the side that the sum leaves out), and of two chunks
    float *near = walk.wu + W::C, *far = near + 64;
    if (tid < 64) {
        const int d = J.rev ? tid - 31 : 31 - tid;
        near[tid] = d >= 0 ? J.amul * power(at.a2, d) : 0.f;
    } else if (tid < 128) {
        far[tid - 64] = J.amul * power(at.a2, J.rev ? tid - 63 : 127 - tid);
    }
    bf16x8* slot = reinterpret_cast<bf16x8*>(smem + W::LDS + 64 * 4) + wb * AT * 2 * 64 + lane;         // [2][NB][AT * 2][64]
    constexpr int SLOT = NB * AT * 2 * 64;
    if (carry) {
        f32x16 S[AT];
        const float* src = a.G > 1 ? J.seg + (at.nh * a.G + at.seg) * E : (J.init ? J.init + at.nh * E : nullptr);
        const bool turned = a.G == 1 && J.init_t;
#pragma unroll
        for (int x = 0; x < AT; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * x + tile_row(r, h);
                S[x][r] = src && row < J.da && b < J.db ? src[turned ? b * J.da + row : row * J.db + b] : 0.f;
            }
        for (int t = 0; t < walk.nc; ++t) {
#pragma unroll
            for (int x = 0; x < 2 * AT; ++x) slot[(t & 1) * SLOT + 64 * x] = tile_frag<T>(S[x >> 1], x & 1);
            const int m = walk.put(set, t, tid);
            walk.fetch(set, t + 1);
#pragma unroll 1
            for (int u = 0; u < 2; ++u) {
                const int it = walk.rev ? 1 - u : u, mi = min(32, m - 32 * it);
                if (mi <= 0) continue;
                typename Ty<T>::Frag zf[2];
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) zf[kb] = col_frag<W::PB>(walk.Zs, 32 * it + 16 * kb, 32 * wb, lane);
                absorb<T, W::PA, AT, (EXACT ? 3 : 2)>(S, walk.Ys, walk.wu, zf, power(at.a2, mi), it, lane);
            }
        }
        if (EXACT && J.last && b < J.db)
#pragma unroll
            for (int x = 0; x < AT; ++x)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int row = 32 * x + tile_row(r, h);
                    if (row < J.da) J.last[at.nh * E + row * J.db + b] = S[x][r];
                }
    } else {
        const int diag = 31 + 4 * h - l31;
        const float imul = J.imul;
        const int64_t ostep = J.so.s;
        const int db = J.db;
        for (int t = 0; t < walk.nc; ++t) {
            const int t0 = at.s0 + W::C * walk.tile(t), m = walk.put(set, t, tid);
            walk.fetch(set, t + 1);
#pragma unroll 1
            for (int u = 0; u < 2; ++u) {
                const int it = walk.rev ? 1 - u : u, mi = min(32, m - 32 * it);
                if (mi <= 0) continue;
                const T* xr = walk.Xs + (32 * it + l31) * W::PA;
                f32x16 o = zero16();
#pragma unroll
                for (int y = 0; y < AT; ++y)
#pragma unroll
                    for (int k2 = 0; k2 < 2; ++k2) o = mul(slot[(t & 1) * SLOT + 64 * (2 * y + k2)], spread_frag(xr + 32 * y + 16 * k2 + 4 * h), o);
                const float wi = imul * power(at.a2, walk.rev ? max(m - 1 - 32 * it - l31, 0) : 32 * it + l31 + 1);
#pragma unroll
                for (int r = 0; r < 16; ++r) o[r] *= wi;
                auto meet = [&](int jt, const float* decay) {                    // the tokens of half jt
                    const T* yr = walk.Ys + (32 * jt + l31) * W::PA;
                    f32x16 x = zero16();
#pragma unroll
                    for (int k = 0; k < KA; ++k) x = mul(near_frag(yr + 16 * k + 8 * h), near_frag(xr + 16 * k + 8 * h), x);
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] *= decay[tile_row(r, 0)];
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) o = mul(col_frag<W::PB>(walk.Zs, 32 * jt + 16 * kb, 32 * wb, lane), tile_frag<T>(x, kb), o);
                };
                meet(it, near + diag);
                if (u && m > 32) meet(1 - it, far + diag);
                if (l31 < mi) {
                    T* row = op + (t0 + 32 * it + l31) * ostep;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int col = 32 * wb + 8 * q + 4 * h;
                        store4<VEC>(row + col, f32x4{o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]}, db - col);
                    }
                }
            }
        }
    }
    // rows behind the sequence's length
    for (int x = tid; x < (at.send - at.s1) * J.db; x += NT) {
        const int row = x / J.db;
        op[(int64_t)(at.s1 + row) * J.so.s + (x - row * J.db)] = (T)0.f;
    }
}

// ---------------------------------------------------------------- one token
// a workgroup per head: 16-byte pieces of the state's rows over the threads, the row sums meet through LDS in row-group order.
// Bound by reading and writing the state: 512 x 12 heads of 64 x 64 in 38 us, 5.3 TB/s (a large copy: 4.9); 12 heads of 25: 4 us.
template <class T, bool VEC>
__global__ __launch_bounds__(256) void lin_step_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                       const float* __restrict__ log_decay, const float* state, int H, int dk, int dv, int lanes,
                                                       float scale, T* __restrict__ out, float* out_state) {
    constexpr int E = VEC ? 4 : 1;
    __shared__ float part[256 * E];
    const int64_t nh = blockIdx.x;
    const int h = (int)(nh % H), groups = 256 / lanes, col = (threadIdx.x % lanes) * E, grp = threadIdx.x / lanes;
    const float w = __builtin_amdgcn_exp2f(log_decay[h] * al::LOG2E);
    const float* src = state + nh * dk * dv;
    float* dst = out_state + nh * dk * dv;
    const int c0 = col;
    if (c0 < dv) {                                           // lanes * E >= dv
        float vv[E], o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) { vv[e] = (float)v[nh * dv + c0 + e]; o[e] = 0.f; }
#pragma unroll 4
        for (int r = grp; r < dk; r += groups) {
            const float kr = (float)k[nh * dk + r], qr = (float)q[nh * dk + r];
            float s[E];
            if (VEC) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(src + r * dv + c0);
#pragma unroll
                for (int e = 0; e < E; ++e) s[e] = x[e];
            } else s[0] = src[r * dv + c0];
#pragma unroll
            for (int e = 0; e < E; ++e) { s[e] = fmaf(w, s[e], kr * vv[e]); o[e] = fmaf(qr, s[e], o[e]); }
            if (VEC) *reinterpret_cast<f32x4*>(dst + r * dv + c0) = f32x4{s[0], s[E > 1 ? 1 : 0], s[E > 2 ? 2 : 0], s[E > 3 ? 3 : 0]};
            else dst[r * dv + c0] = s[0];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) part[threadIdx.x * E + e] = o[e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < dv; c += 256) {
        const int lane = c / E, e = c % E;
        float o = 0.f;
        for (int g = 0; g < groups; ++g) o += part[(g * lanes + lane) * E + e];
        out[nh * dv + c] = (T)(o * scale);
    }
}

// ---------------------------------------------------------------- host
// heads * sequences that leave the chip part empty are cut into segments, down to 256 tokens each, at least three of them, and only past
// 1024 tokens: the extra pass reads y and z again, and a scan follows it.  Sequences of 1000 tokens of 12 heads, whole and in three, us of
// device time, forward / forward and backward: 16 of them, bf16, 64 wide: 34 / 87 and 48 / 101; 4 of them: 33 / 64 and 31 / 71; one: 33 / 63
// and 29 / 58.  Where one wave does everything whole sequences lose there: one, bf16, 128 wide: 78 / 148 and 54 / 114; one, fp32, 25 wide:
// 135 / 267 and 80 / 160 (in eight of 128 tokens: 46 / 95).  2 x 12 of 16384, bf16, in 32: 80 us.  Aimed at as many workgroups as the chip holds
// at once: three per CU of the pair kernel (512 workgroups: 73 us, 768: 69, 1024: 83), four of the other.
static void cut(Args& a, bool bf16) {
    const int64_t blocks = a.jobs * a.N * a.H, aim = bf16 && a.job[0].da <= 64 && a.job[0].db <= 64 ? 768 : 1024;
    a.G = 1; a.per = (a.S + UNIT - 1) / UNIT * UNIT;
    const int64_t want = std::min<int64_t>(blocks > 0 ? aim / blocks : 0, a.S / 256);
    if (want < 3 || a.S <= 1024) return;
    a.per = (int)((((int64_t)a.S + want - 1) / want + UNIT - 1) / UNIT * UNIT);
    a.G = (a.S + a.per - 1) / a.per;
}
static int pad32(int d) { return d <= 32 ? 32 : (d <= 64 ? 64 : 128); }

template <class T, int DA, int DB, bool VEC> static int launch(const Args& a, hipStream_t s) {
    constexpr size_t out_lds = Walk<T, DA, DB, VEC, true>::LDS, state_lds = Walk<T, DA, DB, VEC, false>::LDS;
    const int64_t grid = a.jobs * a.N * a.H * a.G;
    NR_UNSUPPORTED(grid > 0x7fffffff, "linear_attention: %lld workgroups", (long long)grid);
    if (a.G > 1) {
        if (state_lds > 64 * 1024)
            (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&lin_state_kernel<T, DA, DB, VEC>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)state_lds);
        hipLaunchKernelGGL((lin_state_kernel<T, DA, DB, VEC>), dim3((unsigned)grid), dim3(2 * DB), state_lds, s, a);
        if (int rc = check_launch("linear_attention states")) return rc;
        int64_t most = 0;
        for (int j = 0; j < a.jobs; ++j) most = std::max<int64_t>(most, a.N * a.H * (int64_t)(a.job[j].da * a.job[j].db));
        hipLaunchKernelGGL(lin_scan_kernel, dim3((unsigned)((most + 255) / 256), a.jobs), dim3(256), 0, s, a);
        if (int rc = check_launch("linear_attention scan")) return rc;
    }
    bool exact = false;
    for (int j = 0; j < a.jobs; ++j) exact = exact || (a.job[j].last && a.G == 1);
    auto go = [&](auto kernel, int threads, size_t lds) {
        if (lds > 64 * 1024) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, s, a);
        return check_launch("linear_attention");
    };
    if constexpr (sizeof(T) == 2 && PAIRED<DA, DB>) {
        constexpr size_t lds = Walk<T, DA, DB, VEC, true, 4 * DB>::LDS + 64 * 4 + (size_t)2 * DA * DB * 2;
        return exact ? go(&lin_pair_kernel<DA, DB, VEC, true>, 4 * DB, lds) : go(&lin_pair_kernel<DA, DB, VEC, false>, 4 * DB, lds);
    } else {
        return exact ? go(&lin_out_kernel<T, DA, DB, VEC, true>, 2 * DB, out_lds) : go(&lin_out_kernel<T, DA, DB, VEC, false>, 2 * DB, out_lds);
    }
}
template <class T, int DA, bool VEC> static int pick_b(const Args& a, hipStream_t s) {
    const int b = pad32(a.job[0].db);
    return b == 32 ? launch<T, DA, 32, VEC>(a, s) : (b == 64 ? launch<T, DA, 64, VEC>(a, s) : launch<T, DA, 128, VEC>(a, s));
}
template <class T, bool VEC> static int pick_a(const Args& a, hipStream_t s) {
    const int d = pad32(a.job[0].da);
    return d == 32 ? pick_b<T, 32, VEC>(a, s) : (d == 64 ? pick_b<T, 64, VEC>(a, s) : pick_b<T, 128, VEC>(a, s));
}
static int run(const Args& a, bool bf16, hipStream_t s) {
    const size_t e = bf16 ? 2 : 4;
    bool vec = true;
    for (int j = 0; j < a.jobs; ++j) {
        const Job& J = a.job[j];
        vec = vec && al::aligned16(J.x, J.sx, J.da, e, UNIT) && al::aligned16(J.y, J.sy, J.da, e, UNIT) && al::aligned16(J.z, J.sz, J.db, e, UNIT) && al::aligned16(J.o, J.so, J.db, e, UNIT);
    }
    return bf16 ? (vec ? pick_a<__bf16, true>(a, s) : pick_a<__bf16, false>(a, s)) : (vec ? pick_a<float, true>(a, s) : pick_a<float, false>(a, s));
}
static Args base(const LinProblem& p) {
    Args a{};
    a.N = p.N; a.S = p.S; a.H = p.H; a.log_decay = p.log_decay; a.lens = p.lens;
    return a;
}
static size_t seg_floats(const Args& a) {
    size_t f = 0;
    if (a.G > 1)
        for (int j = 0; j < a.jobs; ++j) f += (size_t)(a.N * a.H) * a.G * a.job[j].da * a.job[j].db;
    return f;
}
static void place_segs(Args& a, float*& ws) {
    if (a.G > 1)
        for (int j = 0; j < a.jobs; ++j) { a.job[j].seg = ws; ws += (size_t)(a.N * a.H) * a.G * a.job[j].da * a.job[j].db; }
}
static AttnStrides dense(int S, int H, int d) { return {(int64_t)S * H * d, (int64_t)H * d, d}; }

static Args fwd_args(const LinProblem& p, void* out, float* last) {
    Args a = base(p);
    a.jobs = 1;
    a.job[0] = Job{p.q, p.k, p.v, p.sq, p.sk, p.sv, dense(p.S, p.H, p.dv), out, p.state, 0, last, nullptr, p.dk, p.dv, 0, p.scale, p.scale, 1.f};
    cut(a, p.bf16);
    return a;
}
// the three products of the backward: one launch, or two where dk and dv are padded to different widths
static int bwd_args(const LinProblem& p, const void* g, const float* dlast, void* dq, void* dk, void* dv, float* dstate, Args (&a)[2]) {
    const AttnStrides sg = dense(p.S, p.H, p.dv), sk = dense(p.S, p.H, p.dk);
    const Job jq{g, p.v, p.k, sg, p.sv, p.sk, sk, dq, p.state, 1, nullptr, nullptr, p.dv, p.dk, 0, p.scale, p.scale, 1.f};
    const Job jk{p.v, g, p.q, p.sv, sg, p.sq, sk, dk, dlast, 1, nullptr, nullptr, p.dv, p.dk, 1, p.scale, 1.f, p.scale};
    const Job jv{p.k, p.q, g, p.sk, p.sq, sg, sg, dv, dlast, 0, dstate, nullptr, p.dk, p.dv, 1, p.scale, 1.f, p.scale};
    a[0] = a[1] = base(p);
    a[0].job[0] = jq; a[0].job[1] = jk; a[0].jobs = 2;
    if (pad32(p.dk) == pad32(p.dv)) {
        a[0].job[2] = jv; a[0].jobs = 3;
        cut(a[0], p.bf16);
        return 1;
    }
    a[1].job[0] = jv; a[1].jobs = 1;
    cut(a[0], p.bf16);
    cut(a[1], p.bf16);
    return 2;
}

}  // namespace lin

size_t lin_fwd_ws_bytes(const LinProblem& p) { return lin::seg_floats(lin::fwd_args(p, nullptr, nullptr)) * 4; }
int lin_fwd(const LinProblem& p, void* out, float* last, void* ws, size_t ws_bytes, hipStream_t s) {
    lin::Args a = lin::fwd_args(p, out, last);
    if (ws_bytes < lin::seg_floats(a) * 4 || (!ws && lin::seg_floats(a))) { set_error("linear_attention_fwd: workspace too small"); return NR_ERR_WORKSPACE; }
    float* w = static_cast<float*>(ws);
    lin::place_segs(a, w);
    return lin::run(a, p.bf16, s);
}
size_t lin_bwd_ws_bytes(const LinProblem& p) {
    lin::Args a[2];
    const int n = lin::bwd_args(p, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, a);
    return (lin::seg_floats(a[0]) + (n == 2 ? lin::seg_floats(a[1]) : 0)) * 4;
}
int lin_bwd(const LinProblem& p, const void* dout, const float* dlast, void* dq, void* dk, void* dv, float* dstate, void* ws, size_t ws_bytes,
            hipStream_t s) {
    lin::Args a[2];
    const int n = lin::bwd_args(p, dout, dlast, dq, dk, dv, dstate, a);
    const size_t need = lin_bwd_ws_bytes(p);
    if (ws_bytes < need || (!ws && need)) { set_error("linear_attention_bwd: workspace too small"); return NR_ERR_WORKSPACE; }
    float* w = static_cast<float*>(ws);
    for (int i = 0; i < n; ++i) {
        lin::place_segs(a[i], w);
        if (int rc = lin::run(a[i], p.bf16, s)) return rc;
    }
    return NR_OK;
}

int lin_step(const void* q, const void* k, const void* v, const float* log_decay, const float* state, int64_t N, int H, int dk, int dv, bool bf16,
             float scale, void* out, float* out_state, hipStream_t s) {
    const int64_t grid = N * H;
    NR_UNSUPPORTED(grid > 0x7fffffff, "linear_attention_step: %lld heads", (long long)grid);
    const bool vec = dv % 4 == 0 && ((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(out_state)) & 15) == 0;
    int lanes = 8;                                           // threads along a row of the state
    while (lanes * (vec ? 4 : 1) < dv) lanes *= 2;
#define NR_STEP(T, VEC) hipLaunchKernelGGL((lin::lin_step_kernel<T, VEC>), dim3((unsigned)grid), dim3(256), 0, s, static_cast<const T*>(q), \
        static_cast<const T*>(k), static_cast<const T*>(v), log_decay, state, H, dk, dv, lanes, scale, static_cast<T*>(out), out_state)
    if (bf16) { if (vec) NR_STEP(__bf16, true); else NR_STEP(__bf16, false); }
    else      { if (vec) NR_STEP(float, true); else NR_STEP(float, false); }
#undef NR_STEP
    return check_launch("linear_attention_step");
}

}  // namespace nr
