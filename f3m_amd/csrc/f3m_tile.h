// Tiles of the kernel products over sequences: element types, fragments of the matrix instructions, LDS layouts.
//
// All products run on 32x32 tiles with 16 inner indices per step.  Lane l of a wavefront (half h = l / 32) supplies row
// (of A) or column (of B) l % 32 for the eight inner indices 8h..8h+7 and holds, in element r of the result,
// D[8(r/4) + 4h + r%4][l%32].  If row x of A is taken from source row tile_row(x) (bits 2 and 3 of x swapped), element r
// of half h is source row 16(r/8) + 8h + r%8: eight neighbouring elements are then exactly the eight inner indices that
// the same lane supplies to a product over those rows.  The result of one product is so the operand of the next without leaving its lane.
#pragma once
#include "f3m_rt.h"

#include <cmath>

namespace f3m {

#ifdef F3M_CPU_EMU
typedef uint32_t u32x4 __attribute__((vector_size(16)));
typedef uint32_t u32x2 __attribute__((vector_size(8)));
#else
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 hf2 __attribute__((ext_vector_type(2)));
typedef float f2 __attribute__((ext_vector_type(2)));
#endif

__device__ __forceinline__ float as_float(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ __forceinline__ u32x4 zero4() { return u32x4{0u, 0u, 0u, 0u}; }
__device__ __forceinline__ int tile_row(int x) { return (x & ~12) | ((x & 4) << 1) | ((x & 8) >> 1); }

// ---- element types ---------------------------------------------------------------------------------
// pack / unpack: two neighbouring elements of one 32-bit word, each rounded once to nearest even.
struct Bf16 {
    static constexpr int kBytes = 2, kId = 0;
    typedef u32x4 Frag;
#ifdef F3M_CPU_EMU
    static uint32_t one(float f)
    {
        uint32_t u = as_bits(f);
        if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
        return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
    }
    static uint32_t pack(float a, float b) { return one(a) | (one(b) << 16); }
#else
    __device__ static __forceinline__ uint32_t pack(float a, float b)
    {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), bf2));
    }
#endif
    __device__ static __forceinline__ float lo(uint32_t u) { return as_float(u << 16); }
    __device__ static __forceinline__ float hi(uint32_t u) { return as_float(u & 0xffff0000u); }
};
struct Fp16 {
    static constexpr int kBytes = 2, kId = 1;
    typedef u32x4 Frag;
#ifdef F3M_CPU_EMU
    static uint32_t pack(float a, float b) { return to_half(a).bits | ((uint32_t)to_half(b).bits << 16); }
    static float lo(uint32_t u) { return half_to_float(half_t{(uint16_t)(u & 0xffffu)}); }
    static float hi(uint32_t u) { return half_to_float(half_t{(uint16_t)(u >> 16)}); }
#else
    __device__ static __forceinline__ uint32_t pack(float a, float b)
    {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), hf2));
    }
    __device__ static __forceinline__ float lo(uint32_t u) { return (float)__builtin_bit_cast(hf2, u)[0]; }
    __device__ static __forceinline__ float hi(uint32_t u) { return (float)__builtin_bit_cast(hf2, u)[1]; }
#endif
};
struct Frag32 { u32x4 v[2]; };
struct Fp32 {
    static constexpr int kBytes = 4, kId = 2;
    typedef Frag32 Frag;
};
template <class T> constexpr int kPer16 = 16 / T::kBytes;       // elements of 16 bytes

// ---- fragments: eight elements of one lane -------------------------------------------------------------
template <class T> __device__ __forceinline__ typename T::Frag to_frag(const float *f)
{
    return u32x4{T::pack(f[0], f[1]), T::pack(f[2], f[3]), T::pack(f[4], f[5]), T::pack(f[6], f[7])};
}
template <> __device__ __forceinline__ Frag32 to_frag<Fp32>(const float *f)
{
    return Frag32{{u32x4{as_bits(f[0]), as_bits(f[1]), as_bits(f[2]), as_bits(f[3])},
                   u32x4{as_bits(f[4]), as_bits(f[5]), as_bits(f[6]), as_bits(f[7])}}};
}
template <class T> __device__ __forceinline__ void from_frag(const typename T::Frag &x, float *f)
{
    for (int i = 0; i < 4; i++) { f[2 * i] = T::lo(x[i]); f[2 * i + 1] = T::hi(x[i]); }
}
template <> __device__ __forceinline__ void from_frag<Fp32>(const Frag32 &x, float *f)
{
    for (int i = 0; i < 8; i++) f[i] = as_float(x.v[i >> 2][i & 3]);
}
template <class T> __device__ __forceinline__ typename T::Frag zero_frag() { return zero4(); }
template <> __device__ __forceinline__ Frag32 zero_frag<Fp32>() { return Frag32{{zero4(), zero4()}}; }

// f[8] as a sum of NS fragments, the rest of each rounding in the next
template <class T, int NS> __device__ __forceinline__ void split_frag(const float *f, typename T::Frag *out)
{
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; e++) rest[e] = f[e];
#pragma unroll
    for (int n = 0; n < NS; n++) {
        out[n] = to_frag<T>(rest);
        if (n + 1 < NS) {
            float got[8];
            from_frag<T>(out[n], got);
#pragma unroll
            for (int e = 0; e < 8; e++) rest[e] -= got[e];
        }
    }
}

// 2^n, n from -126 to 127; 0 below, 2^127 above
__device__ __forceinline__ float power_of_two(int n) { return as_float(n < -126 ? 0u : (uint32_t)(127 + (n > 127 ? 127 : n)) << 23); }
// n with 2^n <= x < 2^(n+1), taken into -100 .. 127: 2^(13 - n) and its inverse are then normal numbers
__device__ __forceinline__ int exponent_of(float x)
{
    const int n = (int)(as_bits(x) >> 23) - 127;
    return n < -100 ? -100 : n > 127 ? 127 : n;
}

// largest magnitude of n fragments of fp16: without the sign they are ordered as 16-bit numbers are
__device__ __forceinline__ float largest(const u32x4 *x, int n)
{
#ifdef F3M_CPU_EMU
    float top = 0.f;
    for (int i = 0; i < n; i++)
        for (int j = 0; j < 4; j++) top = fmaxf(top, fmaxf(fabsf(Fp16::lo(x[i][j])), fabsf(Fp16::hi(x[i][j]))));
    return top;
#else
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    us2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < n; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, x[i][j] & 0x7fff7fffu));
    const uint32_t u = __builtin_bit_cast(uint32_t, top);
    return fmaxf(Fp16::lo(u), Fp16::hi(u));
#endif
}

// c += A B over the sixteen inner indices of one step
#ifdef F3M_CPU_EMU
template <class T> inline f32x16 mma(const typename T::Frag &a, const typename T::Frag &b, f32x16 c, int site = __builtin_LINE())
{
    float fa[8], fb[8];
    from_frag<T>(a, fa);
    from_frag<T>(b, fb);
    uint32_t A[8][64], B[8][64];
    for (int e = 0; e < 8; e++) { emu::gather_bits(as_bits(fa[e]), A[e], site); emu::gather_bits(as_bits(fb[e]), B[e], site); }
    const unsigned l = lane_id(), j = l & 31, h = l >> 5;
    for (int r = 0; r < 16; r++) {
        const unsigned i = 8 * (r / 4) + 4 * h + (r % 4);
        double acc = c.v[r];
        for (int hh = 0; hh < 2; hh++)
            for (int e = 0; e < 8; e++) acc += (double)as_float(A[e][i + 32 * hh]) * (double)as_float(B[e][j + 32 * hh]);
        c.v[r] = (float)acc;
    }
    return c;
}
#else
template <class T> __device__ __forceinline__ f32x16 mma(const typename T::Frag &a, const typename T::Frag &b, f32x16 c);
template <> __device__ __forceinline__ f32x16 mma<Bf16>(const u32x4 &a, const u32x4 &b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mma<Fp16>(const u32x4 &a, const u32x4 &b, f32x16 c)
{
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
// the fp32 instruction takes two inner indices, one per half: the eight of a lane in eight instructions
template <> __device__ __forceinline__ f32x16 mma<Fp32>(const Frag32 &a, const Frag32 &b, f32x16 c)
{
#pragma unroll
    for (int e = 0; e < 8; e++)
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(as_float(a.v[e >> 2][e & 3]), as_float(b.v[e >> 2][e & 3]), c, 0, 0, 0);
    return c;
}
#endif
__device__ __forceinline__ f32x16 zero_acc()
{
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; r++) z[r] = 0.f;
    return z;
}
// sum and maximum over the two lanes that share a column
#ifdef F3M_CPU_EMU
inline float half_max(float x, int site = __builtin_LINE()) { return fmaxf(x, wave_shfl_xor_f(x, 32, site)); }
inline float half_sum(float x, int site = __builtin_LINE()) { return x + wave_shfl_xor_f(x, 32, site); }
#else
__device__ __forceinline__ float half_max(float x)
{
    const auto p = __builtin_amdgcn_permlane32_swap(as_bits(x), as_bits(x), false, false);    // both halves' values, in both halves
    return fmaxf(as_float(p[0]), as_float(p[1]));
}
__device__ __forceinline__ float half_sum(float x)
{
    const auto p = __builtin_amdgcn_permlane32_swap(as_bits(x), as_bits(x), false, false);
    return as_float(p[0]) + as_float(p[1]);
}
#endif

// ---- LDS tiles -------------------------------------------------------------------------------------------
// Row-major, in units of 16 bytes.  A fragment along a row is one 16-byte read a lane; a fragment down a column is two transposing reads of 8
// bytes (ds_read_b64_tr_b16: sixteen lanes read a block of 4 rows x 16 columns and get it back by columns), for fp32 eight reads of
// one element.  LDS has 64 banks, sixteen units wide: sixteen lanes read sixteen rows at one unit, thirty-two read four rows at four units.  Unit
// u of row r lies at u ^ swizzle(r), which gives sixteen rows sixteen different places and the four rows of a
// transposing read places apart from each other (padding the rows serves one of the two reads, not both: 10 cycles a fragment instead of 6).
template <class T, int W> constexpr int kRowUnits = W / kPer16<T> == 12 ? 16 : W / kPer16<T> == 24 ? 32 : W / kPer16<T>;
template <int U> __device__ __forceinline__ int swizzle(int r)
{
    if constexpr (U >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (U == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
}

#ifdef F3M_CPU_EMU
inline u32x2 transposed_read(const u32x2 *p, int site = __builtin_LINE())
{
    uint32_t w[2][64];
    emu::gather_bits((*p)[0], w[0], site);
    emu::gather_bits((*p)[1], w[1], site);
    const unsigned l = lane_id(), j = l & 15;
    uint16_t e[4];
    for (unsigned k = 0; k < 4; k++) {
        const uint32_t v = w[(j & 3) >> 1][(l & ~15u) + 4 * k + j / 4];
        e[k] = (uint16_t)(j & 1 ? v >> 16 : v);
    }
    return u32x2{e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16};
}
#else
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ u32x2 transposed_read(const u32x2 *p)
{
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p));
}
#endif

template <class T, int W> struct Tile {
    static constexpr int U = kRowUnits<T, W>;
    // A lane's part of the address of a fragment read: the same for all tiles, rows of 16 and pieces of a row, which change it by an offset and by
    // an exclusive-or with a constant.
    // along a row: the eight elements from 16 n + 8 h of row base + r (base a multiple of 16)
    __device__ static __forceinline__ int row_lane(int r, int h) { return r * U + ((T::kBytes == 2 ? h : 2 * h) ^ swizzle<U>(r)); }
    __device__ static __forceinline__ typename T::Frag row(const u32x4 *tile, int base, int lane, int n)
    {
        const u32x4 *p = tile + base * U;
        if constexpr (T::kBytes == 2) return p[lane ^ (2 * n)];
        else return Frag32{{p[lane ^ (4 * n)], p[lane ^ (4 * n + 1)]}};
    }
    // down a column: elements of the eight rows from base + 8 h in column 32 n + l, or 32 n + tile_row(l) if swapped (l = lane % 32, h = lane / 32)
    struct ColLane { int a, b; };
    __device__ static __forceinline__ ColLane col_lane(int l, int h, bool swapped = false)
    {
        if constexpr (T::kBytes == 2) {
            const int four = swapped ? ((l & 1) << 1) | ((l >> 1) & 1) : l & 3;     // which four of the block's columns this lane reads
            const int r = 8 * h + ((l >> 2) & 3), u = 2 * (l >> 4) + (four >> 1);
            return ColLane{r * (2 * U) + (four & 1) + 2 * (u ^ swizzle<U>(r)), (r + 4) * (2 * U) + (four & 1) + 2 * (u ^ swizzle<U>(r + 4))};
        } else return ColLane{swapped ? tile_row(l) : l, h};
    }
    __device__ static __forceinline__ typename T::Frag col(const u32x4 *tile, int base, ColLane lane, int n)
    {
        if constexpr (T::kBytes == 2) {
            const u32x2 *p = reinterpret_cast<const u32x2 *>(tile) + base * (2 * U);
            const u32x2 a = transposed_read(p + (lane.a ^ (8 * n))), b = transposed_read(p + (lane.b ^ (8 * n)));
            return u32x4{a[0], a[1], b[0], b[1]};
        } else {
            const int c = 32 * n + lane.a;
            const uint32_t *p = reinterpret_cast<const uint32_t *>(tile) + (base + 8 * lane.b) * (4 * U) + (c & 3);
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = p[e * (4 * U) + 4 * ((c >> 2) ^ swizzle<U>(8 * lane.b + e))];
            return Frag32{{u32x4{w[0], w[1], w[2], w[3]}, u32x4{w[4], w[5], w[6], w[7]}}};
        }
    }
    __device__ static __forceinline__ void put(u32x4 *tile, u32x4 x, int row, int c) { tile[row * U + (c ^ swizzle<U>(row))] = x; }
};

// The same value, which the compiler may not compute with outside the loop: what it derives from it (addresses) is computed
// where it is used and takes no registers over the loop.
#ifdef F3M_CPU_EMU
inline int in_loop(int lane_value) { return lane_value; }
#else
__device__ __forceinline__ int in_loop(int lane_value)
{
    asm volatile("" : "+v"(lane_value));
    return lane_value;
}
#endif

// Waits for a fragment that was loaded before a loop: used first inside, it would be waited for there, together with the loop's own loads.
template <class F> __device__ __forceinline__ void settle(F &x)
{
#ifndef F3M_CPU_EMU
    if constexpr (sizeof(F) == 16) asm volatile("" : "+v"(x));
    else { asm volatile("" : "+v"(x.v[0])); asm volatile("" : "+v"(x.v[1])); }
#endif
}

// Order of issue inside a straight piece of code: n LDS reads (n matrix instructions) next.  The compiler by itself reads a fragment just
// before its use and waits for it.
#ifdef F3M_CPU_EMU
#define F3M_NEXT_READS(n)
#define F3M_NEXT_MMA(n)
#define F3M_FENCE()
#else
#define F3M_NEXT_READS(n) __builtin_amdgcn_sched_group_barrier(0x100, n, 0)
#define F3M_NEXT_MMA(n) __builtin_amdgcn_sched_group_barrier(0x8, n, 0)
// Instructions stay on their side of this point (the order above gives way where registers are short).
#define F3M_FENCE() __builtin_amdgcn_sched_barrier(0)
#endif

// Order of N matrix instructions that take READS LDS reads each: those of AHEAD instructions are under way before their uses, after FIRST other reads.
template <int N, int READS, int AHEAD, int FIRST = 0> __device__ __forceinline__ void read_ahead()
{
    F3M_NEXT_READS(FIRST + AHEAD * READS);
#pragma unroll
    for (int n = 0; n < N - AHEAD; n++) { F3M_NEXT_MMA(1); F3M_NEXT_READS(READS); }
    F3M_NEXT_MMA(AHEAD);
}

// ---- global loads without branches ----------------------------------------------------------------------
// 16 bytes at base + offset if they end within `bytes`, else zero (the bounds check of the buffer instructions).
constexpr int kOutside = 0x7fffffe0;
#ifdef F3M_CPU_EMU
struct Buffer { const char *base; int bytes; };
inline Buffer buffer(const void *base, int bytes) { return Buffer{(const char *)base, bytes}; }
inline u32x4 load16(const Buffer &b, int offset)
{
    if ((uint32_t)offset + 16u > (uint32_t)b.bytes) return zero4();
    return *reinterpret_cast<const u32x4 *>(b.base + offset);
}
#else
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer(const void *base, int bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, bytes, 0x00027000);
}
__device__ __forceinline__ u32x4 load16(Buffer b, int offset)
{
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(b, offset, 0, 0));
}
#endif

// writes n (a multiple of 4) neighbouring elements of one row, fp32 values rounded once
template <class T> __device__ __forceinline__ void store4(void *row, int e, float a, float b, float c, float d)
{
    if constexpr (T::kBytes == 2) *reinterpret_cast<u32x2 *>(static_cast<char *>(row) + 2 * e) = u32x2{T::pack(a, b), T::pack(c, d)};
    else *reinterpret_cast<u32x4 *>(static_cast<char *>(row) + 4 * e) = u32x4{as_bits(a), as_bits(b), as_bits(c), as_bits(d)};
}

// Workgroups are dealt to the eight XCDs in turn.  This order gives each XCD a contiguous run of items, so that items that read the same
// keys share an L2.  Returns n or more for the workgroups that pad the last run.
__device__ __forceinline__ int xcd_item(int block, int n)
{
    const int per = (n + 7) / 8;
    const int at = (block & 7) * per + (block >> 3);
    return (block >> 3) < per ? at : n;
}
inline unsigned xcd_grid(long long n) { return (unsigned)(8 * ((n + 7) / 8)); }

// ---- C ABI plumbing --------------------------------------------------------------------------------------
// Entry points that queue their kernels and return: an error is reported and nothing is waited for.
template <typename F> int guarded_async(F f)
{
    try {
        f();
        return 0;
    } catch (const Error &e) {
        g_error = e.what();
        return e.code;
    } catch (const std::exception &e) {
        g_error = e.what();
        return 99;
    } catch (...) {
        g_error = "unknown exception";
        return 99;
    }
}
inline void check_16(const void *p, const char *name)
{
    F3M_REQUIRE(p != nullptr, 8, "%s is NULL", name);
    F3M_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0, 60, "%s is not aligned to 16 bytes", name);
}
inline void check_strides(const int64_t *s, int bytes, const char *name)
{
    for (int i = 0; i < 3; i++)
        F3M_REQUIRE((s[i] * bytes) % 16 == 0, 60, "stride %d of %s (%lld elements) is not a multiple of 16 bytes", i, name, (long long)s[i]);
}
// calls f with the element type
template <typename F> void with_type(int dtype, F f)
{
    if (dtype == Bf16::kId) f(Bf16{});
    else if (dtype == Fp16::kId) f(Fp16{});
    else f(Fp32{});
}

}  // namespace f3m
