// 32x32 matrix-core tiles over one element type, for kernels that run the same tiling on fp32 and on bf16 tensors
// (attention_long.hip, linear_attention.hip).
//
// A product D[i][j] += sum_k A[i][k] B[k][j] is taken in k-steps of 16.  A lane (l = lane & 31, h = lane >> 5) holds 8 of the 16
// k's of row i = l of A and of column j = l of B ("fragment"), and 16 elements of D: column j = l, rows
// row(r, h) = (r & 3) + 8 * (r >> 2) + 4 * h.  WHICH 8 of the k's a lane half holds is free as long as A and B agree; two orders
// are used:
//   "near":  k = 8 h + e                        (operands read as 8 consecutive elements of a row)
//   "tile":  k = 4 h + (e & 3) + 8 * (e >> 2)   (operands that are D tiles of an earlier product: element e of k-step kb is
//                                                register 8 kb + e, so a D tile feeds the next product without leaving the lane)
// Element types M of the products:
//   __bf16  one v_mfma_f32_32x32x16_bf16 per k-step
//   Split3  fp32 operands as the sum of three bf16 numbers each (exact: 24 bits in three eights); of the nine partial products the six
//           largest, smallest first, on the bf16 matrix pipe, summed in fp32, at 6 / 16 of the matrix time.  The parts are cut off, not
//           rounded: the second is below 2^-7 and the third below 2^-15 of the operand's power of two, and what is left out below
//           2^-21 of the product, 2^-24.5 on average, always towards zero.  (Rounded parts leave out 2^-24 at most, to both sides, but
//           turn what is within 2^-8 of fp32's largest into infinities; 32 x 12 histories of 200 x 25: o 2.2e-7 off instead of 2.4e-7,
//           4096 x 64 forward 369 us instead of 364.)  An infinite operand comes out as NaN.
//   float   eight v_mfma_f32_32x32x2_f32, the e-th on element e of both fragments (its two k's are the halves' e-th elements); where
//           memory or latency bounds the kernel and the split would only cost registers
#pragma once
#include "common.h"

namespace nr {
namespace mma {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Split3 {};
struct Frag3 { bf16x8 p[3]; };                   // largest part first

template <class T> struct Ty;
template <> struct Ty<Split3> { typedef Frag3 Frag; };
template <> struct Ty<float> {
    typedef f32x8 Frag;
    static constexpr int E = 4;        // elements per 16 bytes
    static constexpr int PAD = 4;      // LDS pitch = padded width + PAD: 16-byte rows whose starts walk over the banks
};
template <> struct Ty<__bf16> {
    typedef bf16x8 Frag;
    static constexpr int E = 8;
    static constexpr int PAD = 8;
};

__device__ __forceinline__ int tile_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}

__device__ __forceinline__ f32x16 mul(const bf16x8& a, const bf16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mul(const f32x8& a, const f32x8& b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ f32x16 mul(const Frag3& a, const Frag3& b, f32x16 c) {
    c = mul(a.p[2], b.p[0], c);
    c = mul(a.p[0], b.p[2], c);
    c = mul(a.p[1], b.p[1], c);
    c = mul(a.p[1], b.p[0], c);
    c = mul(a.p[0], b.p[1], c);
    return mul(a.p[0], b.p[0], c);
}
// two floats -> their three parts, packed in pairs (x in the low halves)
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& p0, uint32_t& p1, uint32_t& p2) {
    p0 = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
    x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
    p1 = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
    x -= __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    y -= __uint_as_float(__float_as_uint(y) & 0xffff0000u);
    p2 = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
}
__device__ __forceinline__ Frag3 split8(const f32x8& v) {
    u32x4 a, b, c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        uint32_t x, y, z;
        split_pair(v[2 * e], v[2 * e + 1], x, y, z);
        a[e] = x; b[e] = y; c[e] = z;
    }
    return Frag3{{__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, c)}};
}
// a fragment as loaded from memory -> as multiplied
template <class M> struct As;
template <> struct As<__bf16> { static __device__ __forceinline__ bf16x8 frag(const bf16x8& v) { return v; } };
template <> struct As<float> { static __device__ __forceinline__ f32x8 frag(const f32x8& v) { return v; } };
template <> struct As<Split3> { static __device__ __forceinline__ Frag3 frag(const f32x8& v) { return split8(v); } };

// 8 consecutive elements of an LDS row ("near" order: p already points at column 16 * kstep + 8 * h)
__device__ __forceinline__ bf16x8 near_frag(const __bf16* p) { return *reinterpret_cast<const bf16x8*>(p); }
__device__ __forceinline__ f32x8 near_frag(const float* p) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// column col0 + l of the LDS tile, rows row0 + ("tile" order).  bf16: two transposed 8-byte reads, each handing lane i of a
// 16-lane group column i of a 4-row block whose rows the group's lanes 4 q + p address (row q, columns 4 p ..): EXEC must be
// all ones.
template <int PITCH>
__device__ __forceinline__ bf16x8 col_frag(const __bf16* tile, int row0, int col0, int lane) {
    const int g = lane >> 4, q = (lane & 15) >> 2, p = lane & 3;
    const __bf16* z = tile + (row0 + 4 * (g >> 1) + q) * PITCH + col0 + 16 * (g & 1) + 4 * p;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(z));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(z + 8 * PITCH));
    return __builtin_bit_cast(bf16x8, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
}
template <int PITCH>
__device__ __forceinline__ f32x8 col_frag(const float* tile, int row0, int col0, int lane) {
    const float* z = tile + (row0 + 4 * (lane >> 5)) * PITCH + col0 + (lane & 31);
    return f32x8{z[0], z[PITCH], z[2 * PITCH], z[3 * PITCH], z[8 * PITCH], z[9 * PITCH], z[10 * PITCH], z[11 * PITCH]};
}

// two floats rounded to bf16 (to nearest even), the first in the low half
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
// registers 8 kb .. 8 kb + 7 of a D tile as a fragment in "tile" order (bf16: rounded to nearest even)
template <class T> __device__ __forceinline__ typename Ty<T>::Frag tile_frag(const f32x16& t, int kb) {
    typename Ty<T>::Frag o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (T)t[8 * kb + e];
    return o;
}

template <> __device__ __forceinline__ Frag3 tile_frag<Split3>(const f32x16& t, int kb) {
    return split8(f32x8{t[8 * kb], t[8 * kb + 1], t[8 * kb + 2], t[8 * kb + 3], t[8 * kb + 4], t[8 * kb + 5], t[8 * kb + 6], t[8 * kb + 7]});
}

// A [ROWS x D] tile in LDS, to be multiplied as M.  put: 16 bytes of a row as they come from memory
template <class M, int ROWS, int D> struct Lds {
    static constexpr int PITCH = D + Ty<M>::PAD;
    static constexpr size_t BYTES = (size_t)ROWS * PITCH * sizeof(M);
    static __device__ __forceinline__ void put(char* t, int row, int col, const u32x4& v) {
        *reinterpret_cast<u32x4*>(reinterpret_cast<M*>(t) + row * PITCH + col) = v;
    }
    static __device__ __forceinline__ typename Ty<M>::Frag near(const char* t, int row, int col) {
        return near_frag(reinterpret_cast<const M*>(t) + row * PITCH + col);
    }
    static __device__ __forceinline__ typename Ty<M>::Frag col(const char* t, int row0, int col0, int lane) {
        return col_frag<PITCH>(reinterpret_cast<const M*>(t), row0, col0, lane);
    }
};
// the three parts as three bf16 tiles
template <int ROWS, int D> struct Lds<Split3, ROWS, D> {
    typedef Lds<__bf16, ROWS, D> L;
    static constexpr int PITCH = L::PITCH;
    static constexpr size_t BYTES = 3 * L::BYTES;
    static __device__ __forceinline__ void put(char* t, int row, int col, const u32x4& v) {
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        uint32_t a, b, c, d, e, f;
        split_pair(__uint_as_float(v[0]), __uint_as_float(v[1]), a, b, c);
        split_pair(__uint_as_float(v[2]), __uint_as_float(v[3]), d, e, f);
        char* p = t + (row * PITCH + col) * 2;
        *reinterpret_cast<u32x2*>(p) = u32x2{a, d};
        *reinterpret_cast<u32x2*>(p + L::BYTES) = u32x2{b, e};
        *reinterpret_cast<u32x2*>(p + 2 * L::BYTES) = u32x2{c, f};
    }
    static __device__ __forceinline__ Frag3 near(const char* t, int row, int col) {
        return Frag3{{L::near(t, row, col), L::near(t + L::BYTES, row, col), L::near(t + 2 * L::BYTES, row, col)}};
    }
    static __device__ __forceinline__ Frag3 col(const char* t, int row0, int col0, int lane) {
        return Frag3{{L::col(t, row0, col0, lane), L::col(t + L::BYTES, row0, col0, lane), L::col(t + 2 * L::BYTES, row0, col0, lane)}};
    }
};

// E consecutive elements of a global row as one 16-byte word; elements at and past `n` are zero.  VEC: the address is a multiple
// of 16 and n is a multiple of E; otherwise the address is a multiple of the element's size: a whole word is still one load (global
// memory takes 16-byte loads at any address), the end of a row comes element by element.
template <class T, bool VEC>
__device__ __forceinline__ u32x4 load16(const T* p, int n) {
    constexpr int E = Ty<T>::E;
    if (n <= 0) return u32x4{0, 0, 0, 0};
    if (VEC) return *reinterpret_cast<const u32x4*>(p);
    u32x4 o = {0, 0, 0, 0};
    if (n >= E) {
        __builtin_memcpy(&o, p, 16);
        return o;
    }
    if (sizeof(T) == 4) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
        for (int e = 0; e < 3; ++e) if (e < n) o[e] = w[e];
        return o;
    }
    uint32_t s[8];
    const uint16_t* w = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int e = 0; e < 7; ++e) s[e] = e < n ? w[e] : 0;
    return u32x4{s[0] | s[1] << 16, s[2] | s[3] << 16, s[4] | s[5] << 16, s[6]};
}
// a whole fragment (8 consecutive elements, "near" order) from global memory
template <bool VEC> __device__ __forceinline__ bf16x8 load_frag(const __bf16* p, int n) {
    return __builtin_bit_cast(bf16x8, load16<__bf16, VEC>(p, n));
}
template <bool VEC> __device__ __forceinline__ f32x8 load_frag(const float* p, int n) {
    const f32x4 a = __builtin_bit_cast(f32x4, load16<float, VEC>(p, n));
    const f32x4 b = __builtin_bit_cast(f32x4, load16<float, VEC>(p + 4, n - 4));
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
// four consecutive elements (registers 4 i .. 4 i + 3 of a D tile whose rows run along the output's last axis)
template <bool VEC> __device__ __forceinline__ void store4(__bf16* p, const f32x4& v, int n) {
    const bf16x4 o = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    if (VEC) { if (n > 0) *reinterpret_cast<bf16x4*>(p) = o; return; }
    if (n >= 4) { __builtin_memcpy(p, &o, 8); return; }
#pragma unroll
    for (int e = 0; e < 3; ++e) if (e < n) p[e] = o[e];
}
template <bool VEC> __device__ __forceinline__ void store4(float* p, const f32x4& v, int n) {
    if (VEC) { if (n > 0) *reinterpret_cast<f32x4*>(p) = v; return; }
    if (n >= 4) { __builtin_memcpy(p, &v, 16); return; }
#pragma unroll
    for (int e = 0; e < 3; ++e) if (e < n) p[e] = v[e];
}

}  // namespace mma
}  // namespace nr
