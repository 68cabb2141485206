// gsr_adamw.hip -- AdamW over many tensors at once with moments in 32 or in 8 bits, the global
// gradient norm it clips by, and the row selection and conversion of 8-bit moments.
//
// Per element, t the step count after this update and s = grad_scale * clip coefficient:
//     g  = s grad
//     p <- p (1 - lr wd)
//     m <- m + (1 - b1)(g - m)
//     v <- b2 v + (1 - b2) g g
//     p <- p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// A 16-bit parameter has a 32-bit master that takes the update; the parameter is its rounding.
//
// Moments in 8 bits: m and r = sqrt(v) are held as e4m3 codes times a scale for each block of
// 256 consecutive elements of the tensor.  The root halves v's span of exponents, so both
// moments reach from a block's largest value down to 2^-18 of it.  Per block and moment, after
// the update:
//     top = max |x| (finite x), scale = top / 448, y = min(|x| * (1 / top * 448), 448)
//     ulp = 2^(max(floor(log2 y), -6) - 3), code = sign(x) floor(y / ulp + u) ulp
// with u of 16 random bits in [0, 1): the expected code is y.  Rounding to nearest would lose
// what an update changes by less than half a step: v moves by at most 0.1 % of itself when it
// decays, a step is 6 to 12 %, so v (and m for a steady gradient, up to a third of it) would
// stand still.  What is unbiased is the step from one root to the next, not v: a root that moves by
// d of itself, d about c = 1 - b2, and is rounded by steps of s varies by d s more each time, which v
// forgets with c a step and r with c / 2: v is 4 to 8 % too large on average, r 14 to 20 % off.
// u is a function of (seed, tensor, step, element), so a run and every rank
// repeat it exactly.  r > 0 never gets the code 0: v would be lost while m need not be, and
// m / (sqrt(v) + eps) would be m / eps.
//
// Both steps are bound by HBM, at 28 and 16 bytes an element of an fp32 parameter (a copy in place
// of 4 GB reaches 5.9 TB/s on the same card).  Medians of a kernel trace: 23.3M parameters 100 us (6.5 TB/s)
// and 73 us (5.1 TB/s; 62 us, 6.0 TB/s, where calls follow each other untraced), 77.4M with 8-bit moments
// 189 us (6.6 TB/s), 63.5M bf16 ones with masters 262 us (6.8 TB/s).  The 8-bit step's
// two roundings and their hash are about 60 vector instructions an element, which the loads in
// flight of seven waves a SIMD still hide.  Small lists are bound by one launch's latency: 148 K
// elements in 13 tensors 3.8 and 5.4 us.
#include "gsr_adamw.hpp"

namespace gsr {

namespace {

typedef unsigned int u32;

// The rounding of a float.  Without the barrier the compiler joins it with the multiply-add that made
// x, which rounds once instead of twice: a parameter would not be its stored master's rounding.
__device__ __forceinline__ _Float16 to_half(float x) {
    asm volatile("" : "+v"(x));
    return (_Float16)x;
}

__device__ __forceinline__ float load_as_float(const void* p, int type, long long i) {
    if (type == AW_F32) return static_cast<const float*>(p)[i];
    if (type == AW_BF16) return (float)static_cast<const __bf16*>(p)[i];
    return (float)static_cast<const _Float16*>(p)[i];
}

__device__ __forceinline__ void store_from_float(void* p, int type, long long i, float x) {
    if (type == AW_F32)
        static_cast<float*>(p)[i] = x;
    else if (type == AW_BF16)
        static_cast<__bf16*>(p)[i] = (__bf16)x;
    else
        static_cast<_Float16*>(p)[i] = to_half(x);
}

template <int T>
__device__ __forceinline__ float load_as_float(const void* p, long long i) {
    return load_as_float(p, T, i);
}

// Four consecutive elements of type T, T-aligned to 4 elements
template <int T>
struct Vec4;
template <>
struct Vec4<AW_F32> {
    typedef float4 raw;
    static __device__ __forceinline__ float4 get(raw x) { return x; }
    static __device__ __forceinline__ raw put(float4 x) { return x; }
};
template <>
struct Vec4<AW_BF16> {
    typedef __bf16 raw __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ float4 get(raw x) { return make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]); }
    static __device__ __forceinline__ raw put(float4 x) { return raw{(__bf16)x.x, (__bf16)x.y, (__bf16)x.z, (__bf16)x.w}; }
};
template <>
struct Vec4<AW_F16> {
    typedef _Float16 raw __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ float4 get(raw x) { return make_float4((float)x[0], (float)x[1], (float)x[2], (float)x[3]); }
    static __device__ __forceinline__ raw put(float4 x) { return raw{to_half(x.x), to_half(x.y), to_half(x.z), to_half(x.w)}; }
};
template <int T>
__device__ __forceinline__ typename Vec4<T>::raw* vec4(const void* p) {
    return const_cast<typename Vec4<T>::raw*>(static_cast<const typename Vec4<T>::raw*>(p));
}

// What a step reads and writes once and nothing reads before the next one (gradients, moments,
// masters) goes past the caches, which keep the parameters that the next forward reads.  One
// step of three scenes of 23.3M fp32 parameters in turn: 127 us without, 120 with such loads, 100
// with such stores of the moments too (109 where the parameters' stores are like that as well);
// 63M bf16 parameters 328, 309 and 268 us.
typedef float f32x4 __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ T load_once(const T* p) { return __builtin_nontemporal_load(p); }
__device__ __forceinline__ float4 load_once(const float4* p) {
    const f32x4 x = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p));
    return make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void store_once(u32* p, u32 x) { __builtin_nontemporal_store(x, p); }
__device__ __forceinline__ void store_once(float4* p, float4 x) {
    __builtin_nontemporal_store(f32x4{x.x, x.y, x.z, x.w}, reinterpret_cast<f32x4*>(p));
}

// The updated values to the parameter, or to its master and, rounded, to it
template <int PT>
__device__ __forceinline__ void store_parameter(void* param, float4* w, long long q, float4 x) {
    if (PT == AW_F32) {
        *w = x;
    } else {
        store_once(w, x);
        vec4<PT>(param)[q] = Vec4<PT>::put(x);
    }
}

// The last of the tensors whose first group is not behind `group`: first[] ascends, a lane looks at
// one entry.  In arguments:
template <int MAX>
__device__ __forceinline__ int find_tensor(const u32* first, int count, u32 group) {
    int found = 0;
#pragma unroll
    for (int at = 0; at < MAX; at += 64) {
        const int l = at + __lane_id();
        found += __popcll(__ballot(l < count && first[l < MAX ? l : MAX - 1] <= group));
    }
    return __builtin_amdgcn_readfirstlane(found - 1);
}

// The same in memory, of at most 64 * 64: every 64th part of the list first, then the part
__device__ __forceinline__ int find_tensor_in(const u32* __restrict__ first, int count, u32 group) {
    const int part = (count + 63) >> 6;
    const int coarse = __lane_id() * part;
    const int p = __popcll(__ballot(coarse < count && first[coarse < count ? coarse : 0] <= group)) - 1;
    const int l = p * part + __lane_id();
    const bool at = (int)__lane_id() < part && l < count && first[l < count ? l : 0] <= group;
    return __builtin_amdgcn_readfirstlane(p * part + __popcll(__ballot(at)) - 1);
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < INFINITY; }

// One element's update: p, m, v in 32 bits.  No contraction in the moments: what is rounded to 8
// bits afterwards is then the formula's sequence of single roundings, and a code follows from the
// inputs alone, not from how a compiler groups the operations.
__device__ __forceinline__ void update_moments(float g, float& m, float& v, float& root, const AdamWConst& c) {
#pragma clang fp contract(off)
    m = m + c.one_minus_b1 * (g - m);
    const float decayed = c.b2 * v;
    v = decayed + c.one_minus_b2 * (g * g);
    // |g| from 2^64 on: g g is beyond 32 bits, its share in v need not be
    if (__builtin_expect(!is_finite(v), 0)) v = decayed + c.one_minus_b2 * g * g;
    root = sqrtf(v);
}

// The same of m and the root r of v, which 32 bits hold for every finite g: where its square is beyond them it is taken
// of 2^-70 of both, which loses nothing (what is lost beside it is below 2^-100 of it)
__device__ __forceinline__ void update_moments_root(float g, float& m, float& r, const AdamWConst& c) {
#pragma clang fp contract(off)
    m = m + c.one_minus_b1 * (g - m);
    const float v = c.b2 * (r * r) + c.one_minus_b2 * (g * g);
    const float small = r * 0x1p-70f;
    r = sqrtf(v);
    if (__builtin_expect(!is_finite(v), 0)) {
        g = g * 0x1p-70f;
        r = sqrtf(c.b2 * (small * small) + c.one_minus_b2 * (g * g)) * 0x1p70f;
    }
}

__device__ __forceinline__ void update_parameter(float& p, float m, float root, const AdamWConst& c, const AdamWScalars& s) {
    // the reciprocal's error of one unit is the update's, not the moments'
    p = p * s.keep - s.step_size * (m * __builtin_amdgcn_rcpf(root * s.rbc2 + c.eps));
}

// A part of a tensor that is no whole workgroup's, or whose tensors begin at odd places: four
// elements of a thread in flight
template <int PT, int GT>
__device__ __forceinline__ void adamw_scalar(const AdamWTensor& t, const AdamWConst& c, const AdamWScalars& s, float gs,
                                             long long lo, long long hi) {
    float* w = PT == AW_F32 ? static_cast<float*>(t.p) : t.master;
    float* m = static_cast<float*>(t.m);
    float* v = static_cast<float*>(t.v);
    for (long long at = lo + threadIdx.x; at < hi; at += 1024) {
        float P[4], M[4], V[4], G[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const long long i = at + 256 * j;
            if (i >= hi) continue;
            G[j] = load_as_float<GT>(t.g, i);
            P[j] = w[i];
            M[j] = m[i];
            V[j] = v[i];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const long long i = at + 256 * j;
            if (i >= hi) continue;
            float root;
            update_moments(gs * G[j], M[j], V[j], root, c);
            update_parameter(P[j], M[j], root, c, s);
            w[i] = P[j];
            if (PT != AW_F32) store_from_float(t.p, PT, i, P[j]);
            m[i] = M[j];
            v[i] = V[j];
        }
    }
}

// U vectors of four elements a thread: all loads before the first use
template <int PT, int GT, int U>
__device__ __forceinline__ void adamw_vectors(const AdamWTensor& t, const AdamWConst& c, const AdamWScalars& s, float gs,
                                              long long lo) {
    const long long q = (lo >> 2) + threadIdx.x;
    float4* w = reinterpret_cast<float4*>(PT == AW_F32 ? static_cast<float*>(t.p) : t.master) + q;
    float4* m = static_cast<float4*>(t.m) + q;
    float4* v = static_cast<float4*>(t.v) + q;
    const typename Vec4<GT>::raw* g = vec4<GT>(t.g) + q;
    float4 P[U], M[U], V[U];
    typename Vec4<GT>::raw G[U];
#pragma unroll
    for (int j = 0; j < U; j++) {
        G[j] = load_once(g + 256 * j);
        P[j] = load_once(w + 256 * j);
        M[j] = load_once(m + 256 * j);
        V[j] = load_once(v + 256 * j);
    }
#pragma unroll
    for (int j = 0; j < U; j++) {
        const float4 x = Vec4<GT>::get(G[j]);
        float4 root;
        update_moments(gs * x.x, M[j].x, V[j].x, root.x, c);
        update_moments(gs * x.y, M[j].y, V[j].y, root.y, c);
        update_moments(gs * x.z, M[j].z, V[j].z, root.z, c);
        update_moments(gs * x.w, M[j].w, V[j].w, root.w, c);
        update_parameter(P[j].x, M[j].x, root.x, c, s);
        update_parameter(P[j].y, M[j].y, root.y, c, s);
        update_parameter(P[j].z, M[j].z, root.z, c, s);
        update_parameter(P[j].w, M[j].w, root.w, c, s);
        store_parameter<PT>(t.p, w + 256 * j, q + 256 * j, P[j]);
        store_once(m + 256 * j, M[j]);
        store_once(v + 256 * j, V[j]);
    }
}

// The workgroup's 1024 U elements of tensor t, `group` workgroups into it
template <int PT, int GT, int U>
__device__ __forceinline__ void adamw_group(const AdamWTensor& t, const AdamWConst& c, const AdamWScalars& s, float gs,
                                            u32 group) {
    const long long lo = (long long)group * (1024 * U);
    const long long hi = lo + 1024 * U < t.n ? lo + 1024 * U : t.n;
    if (t.aligned && hi - lo == 1024 * U)
        adamw_vectors<PT, GT, U>(t, c, s, gs, lo);
    else
        adamw_scalar<PT, GT>(t, c, s, gs, lo, hi);
}

// ---- 8-bit moments ------------------------------------------------------------------------

__device__ __forceinline__ float decode(u32 code) { return __builtin_amdgcn_cvt_f32_fp8((int)code, 0); }

__device__ __forceinline__ float square(float x) { return x * x; }

__device__ __forceinline__ float finite_abs(float x) { return is_finite(x) ? fabsf(x) : 0.0f; }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}

// A block's largest value -> its scale and what takes a value to its code's range
__device__ __forceinline__ void scales_of(float top, float& scale, float& inv) {
    if (top > 0.0f) {
        top = fmaxf(top, 0x1p-100f);  // 448 / top stays finite
        inv = 1.0f / top * 448.0f;
        scale = top * (1.0f / 448.0f);
    } else {
        inv = scale = 0.0f;
    }
}

// e4m3 code of x: y = |x| inv rounded up with a probability of the part of its step that it is
// over, u16 / 2^16 being the draw.  From 2^-6 on (the least normal) the step is 2^20 units of y's
// bits and the addition carries into the kept ones exactly when part + u >= 1; below, codes
// count steps of 2^-9.
__device__ __forceinline__ u32 encode_random(float x, float inv, u32 u16) {
#pragma clang fp contract(off)
    const float y = fminf(fabsf(x) * inv, 448.0f);
    const u32 high = ((__float_as_uint(y) + (u16 << 4)) >> 20) - 960u;
    const u32 low = (u32)(y * 512.0f + (float)u16 * 0x1p-16f);
    const u32 code = y < 0x1p-6f ? low : high;
    return (is_finite(x) ? code : 0x7fu) | ((__float_as_uint(x) >> 24) & 0x80u);
}

__device__ __forceinline__ u32 root_floor(u32 code, float root) { return root > 0.0f && code == 0 ? 1u : code; }

// A part of a tensor that ends inside a block, or whose tensors begin at odd places: a block of
// 256 elements a wave, lane l having elements l, l + 64, ...
template <int PT, int GT>
__device__ __forceinline__ void adamw8_scalar(const AdamWTensor& t, const AdamWConst& c, const AdamWScalars& s, float gs,
                                              long long lo, long long hi) {
    float* w = PT == AW_F32 ? static_cast<float*>(t.p) : t.master;
    unsigned char* m = static_cast<unsigned char*>(t.m);
    unsigned char* r = static_cast<unsigned char*>(t.v);
    for (long long at = lo + 256 * (threadIdx.x >> 6); at < hi; at += 1024) {
        const long long block = at >> 8;
        const float mscale = t.mscale[block], rscale = t.vscale[block];
        float M[4], R[4], P[4], G[4], mtop = 0.0f, rtop = 0.0f;
        u32 C[4], D[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const long long i = at + 64 * j + __lane_id();
            if (i >= hi) continue;
            C[j] = m[i];
            D[j] = r[i];
            G[j] = load_as_float<GT>(t.g, i);
            P[j] = w[i];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const long long i = at + 64 * j + __lane_id();
            M[j] = R[j] = 0.0f;
            if (i < hi) {
                R[j] = decode(D[j]) * rscale;
                M[j] = decode(C[j]) * mscale;
                update_moments_root(gs * G[j], M[j], R[j], c);
                update_parameter(P[j], M[j], R[j], c, s);
                w[i] = P[j];
                if (PT != AW_F32) store_from_float(t.p, PT, i, P[j]);
            }
            mtop = fmaxf(mtop, finite_abs(M[j]));
            rtop = fmaxf(rtop, finite_abs(R[j]));
        }
        float minv, rinv, mnew, rnew;
        scales_of(wave_max(mtop), mnew, minv);
        scales_of(wave_max(rtop), rnew, rinv);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const long long i = at + 64 * j + __lane_id();
            if (i >= hi) continue;
            const u32 u = aw_mix(s.key + t.first + (u32)i);
            m[i] = (unsigned char)encode_random(M[j], minv, u >> 16);
            r[i] = (unsigned char)root_floor(encode_random(R[j], rinv, u & 0xffffu), R[j]);
        }
        if (__lane_id() == 0) {
            t.mscale[block] = mnew;
            t.vscale[block] = rnew;
        }
    }
}

// The largest of each L consecutive lanes, 32 or 64, in all of them: rotations within rows of 16, then across
template <int L>
__device__ __forceinline__ float lanes_max(float x) {
    static_assert(L == 32 || L == 64, "at least two rows");
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x128, 0xf, 0xf, true)));
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x124, 0xf, 0xf, true)));
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x122, 0xf, 0xf, true)));
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x121, 0xf, 0xf, true)));
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    if (L == 64) x = fmaxf(x, __shfl_xor(x, 32, 64));
    return x;
}

// Whole blocks: L = 64 / U lanes have one, lane l of them the four elements from 4 l of each of the
// block's U parts.  A wave's loads are consecutive within its blocks, the blocks' maxima take five
// or six exchanges, and each thread has 4 U elements in flight.
template <int PT, int GT, int U>
__device__ __forceinline__ void adamw8_vectors(const AdamWTensor& t, const AdamWConst& c, const AdamWScalars& s, float gs,
                                               long long lo) {
    constexpr int L = 64 / U;
    const long long block = (lo >> 8) + threadIdx.x / L;
    const long long q = 64 * block + threadIdx.x % L;
    float4* w = reinterpret_cast<float4*>(PT == AW_F32 ? static_cast<float*>(t.p) : t.master) + q;
    const typename Vec4<GT>::raw* g = vec4<GT>(t.g) + q;
    u32* mc = static_cast<u32*>(t.m) + q;
    u32* rc = static_cast<u32*>(t.v) + q;
    float4 P[U];
    typename Vec4<GT>::raw G[U];
    u32 C[U], D[U];
#pragma unroll
    for (int j = 0; j < U; j++) {
        C[j] = load_once(mc + L * j);
        D[j] = load_once(rc + L * j);
        G[j] = load_once(g + L * j);
        P[j] = load_once(w + L * j);
    }
    const float mscale = t.mscale[block], rscale = t.vscale[block];
    float M[U][4], R[U][4], mtop = 0.0f, rtop = 0.0f;
#pragma unroll
    for (int j = 0; j < U; j++) {
        const float4 x = Vec4<GT>::get(G[j]);
        const float g4[4] = {gs * x.x, gs * x.y, gs * x.z, gs * x.w};
        float p4[4] = {P[j].x, P[j].y, P[j].z, P[j].w};
        M[j][0] = __builtin_amdgcn_cvt_f32_fp8((int)C[j], 0) * mscale;
        M[j][1] = __builtin_amdgcn_cvt_f32_fp8((int)C[j], 1) * mscale;
        M[j][2] = __builtin_amdgcn_cvt_f32_fp8((int)C[j], 2) * mscale;
        M[j][3] = __builtin_amdgcn_cvt_f32_fp8((int)C[j], 3) * mscale;
        R[j][0] = __builtin_amdgcn_cvt_f32_fp8((int)D[j], 0) * rscale;
        R[j][1] = __builtin_amdgcn_cvt_f32_fp8((int)D[j], 1) * rscale;
        R[j][2] = __builtin_amdgcn_cvt_f32_fp8((int)D[j], 2) * rscale;
        R[j][3] = __builtin_amdgcn_cvt_f32_fp8((int)D[j], 3) * rscale;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            update_moments_root(g4[e], M[j][e], R[j][e], c);
            update_parameter(p4[e], M[j][e], R[j][e], c, s);
            mtop = fmaxf(mtop, finite_abs(M[j][e]));
            rtop = fmaxf(rtop, finite_abs(R[j][e]));
        }
        store_parameter<PT>(t.p, w + L * j, q + L * j, make_float4(p4[0], p4[1], p4[2], p4[3]));
    }
    float minv, rinv, mnew, rnew;
    scales_of(lanes_max<L>(mtop), mnew, minv);
    scales_of(lanes_max<L>(rtop), rnew, rinv);
    const u32 key = s.key + t.first + (u32)(4 * q);
#pragma unroll
    for (int j = 0; j < U; j++) {
        u32 c = 0, d = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const u32 u = aw_mix(key + 4 * L * j + e);
            c |= encode_random(M[j][e], minv, u >> 16) << (8 * e);
            d |= root_floor(encode_random(R[j][e], rinv, u & 0xffffu), R[j][e]) << (8 * e);
        }
        store_once(mc + L * j, c);
        store_once(rc + L * j, d);
    }
    if (threadIdx.x % L == 0) {
        t.mscale[block] = mnew;
        t.vscale[block] = rnew;
    }
}

// 4 U blocks
template <int PT, int GT, int U>
__device__ __forceinline__ void adamw8_group(const AdamWTensor& t, const AdamWConst& c, const AdamWScalars& s, float gs,
                                             u32 group) {
    const long long lo = (long long)group * (1024 * U);
    const long long hi = lo + 1024 * U < t.n ? lo + 1024 * U : t.n;
    if (t.aligned && hi - lo == 1024 * U)
        adamw8_vectors<PT, GT, U>(t, c, s, gs, lo);
    else
        adamw8_scalar<PT, GT>(t, c, s, gs, lo, hi);
}

// A gradient norm that is not finite: nothing is changed
__device__ __forceinline__ bool left_out(const AdamWCall& a) { return a.clip && !is_finite(a.clip[0]); }

template <int BITS, int PT, int U>
__device__ __forceinline__ void adamw_by_grad(const AdamWTensor& t, const AdamWConst& c, const AdamWScalars& s, float gs,
                                              u32 group) {
    if (t.grad_type == AW_F32)
        BITS == 8 ? adamw8_group<PT, AW_F32, U>(t, c, s, gs, group) : adamw_group<PT, AW_F32, U>(t, c, s, gs, group);
    else if (t.grad_type == AW_BF16)
        BITS == 8 ? adamw8_group<PT, AW_BF16, U>(t, c, s, gs, group) : adamw_group<PT, AW_BF16, U>(t, c, s, gs, group);
    else
        BITS == 8 ? adamw8_group<PT, AW_F16, U>(t, c, s, gs, group) : adamw_group<PT, AW_F16, U>(t, c, s, gs, group);
}

template <int BITS, int U>
__device__ __forceinline__ void adamw_tensor(const AdamWTensor& t, const AdamWCall& a, const AdamWScalars& s, u32 group) {
    const float gs = a.c.grad_scale * (a.clip ? a.clip[1] : 1.0f);
    if (t.param_type == AW_F32)
        adamw_by_grad<BITS, AW_F32, U>(t, a.c, s, gs, group);
    else if (t.param_type == AW_BF16)
        adamw_by_grad<BITS, AW_BF16, U>(t, a.c, s, gs, group);
    else
        adamw_by_grad<BITS, AW_F16, U>(t, a.c, s, gs, group);
}

template <int BITS, int U>
__global__ void __launch_bounds__(256) k_adamw(AdamWTable a) {
    const int k = find_tensor<AW_TENSORS>(a.first, a.count, blockIdx.x);
    if (left_out(a.call)) return;
    const AdamWTensor t = a.t[k];  // one copy: references into the arguments can move all of them to scratch memory
    const AdamWScalars s = a.call.scalars ? a.call.scalars[a.base + k] : t.s;
    adamw_tensor<BITS, U>(t, a.call, s, blockIdx.x - a.first[k]);
}

// The same over a list in memory (k_adamw_list)
template <int BITS, int U>
__global__ void __launch_bounds__(256) k_adamw_many(AdamWCall a, AdamWRates rates, int count, const u32* __restrict__ first,
                                                    const AdamWTensor* __restrict__ list) {
    const int k = find_tensor_in(first, count, blockIdx.x);
    if (left_out(a)) return;
    const AdamWTensor t = list[k];
    AdamWScalars s = t.s;
    if (a.scalars) {
        s = a.scalars[k];
    } else if (t.rate != AW_OWN) {
        s = rates.r[t.rate & (AW_RATES - 1)];
        s.key = aw_key_at(t.s.key, s.key);
    }
    adamw_tensor<BITS, U>(t, a, s, blockIdx.x - first[k]);
}

// Writes the arguments' tensors to their places in the list in memory
__global__ void __launch_bounds__(256) k_adamw_list(AdamWTable a, u32* __restrict__ first, AdamWTensor* __restrict__ list) {
    static_assert(AW_TENSORS <= 256, "a thread an entry");
    if ((int)threadIdx.x < a.count) first[a.base + threadIdx.x] = a.first[threadIdx.x];
    const u32* from = reinterpret_cast<const u32*>(a.t);
    u32* to = reinterpret_cast<u32*>(list + a.base);
    const int words = a.count * (int)(sizeof(AdamWTensor) / 4);
    for (int i = threadIdx.x; i < words; i += 256) to[i] = from[i];
}

// Steps counted on the device: one thread a tensor advances its count (not when the gradient
// is not finite: that step is left out) and computes what the update takes from it.
__global__ void k_adamw_scalars(AdamWCounts a) {
    const int k = threadIdx.x;
    if (k >= a.count) return;
    const AdamWCount& t = a.t[k];
    if (a.clip && !is_finite(a.clip[0])) return;
    const long long step = *t.step + 1;
    *t.step = step;
    const double lr = t.lr_dev ? (double)*t.lr_dev : t.lr;
    a.scalars[a.base + k] = aw_scalars(step, aw_bias(step, a.b1, a.b2), lr, t.weight_decay, a.seed, t.ordinal);
}

// ---- rows of 8-bit moments ----------------------------------------------------------------

typedef u32 u32_anywhere __attribute__((aligned(1)));

// p[offset / sizeof(T)], the offset in 32 bits: what an address has beside the wave's p
template <typename T>
__device__ __forceinline__ T at_byte(const T* p, u32 offset) {
    return *reinterpret_cast<const T*>(reinterpret_cast<const char*>(p) + offset);
}

// A lane's elements [begin, begin + 4) of the selection, PARTS the most rows that they are of (SINGLE: rows
// of one element): for each part its source (all indices are asked for before the first is used), then both
// moments' codes as words from any address, and their scales; a part that goes on in its row's next block
// has two.  The parts' bytes are put together before they are decoded, and an element's scale is that of the
// last part or block which begins at it or before.  count: how many of the four there are; the others,
// and rows that are not the source's, are zero.  index: the wave's, col, count and `down`, rows from there,
// the lane's.  Place: of a source's elements; 32 bits where they suffice, which is half the
// instructions of the addresses.
template <typename Place, int PARTS, bool SINGLE = false>
__device__ __forceinline__ void gather(const MomentRows& t, const long long* __restrict__ index, u32 down, u32 col, u32 count,
                                       float* x, float* y) {
    const u32 cols = (u32)t.cols;
    long long source[PARTS];
    u32 first[PARTS];
#pragma unroll
    for (int j = 0; j < PARTS; j++) {
        first[j] = j == 0 ? 0u : (u32)j * cols - col;  // count or more: no such part
        source[j] = first[j] < count ? at_byte(index, 8u * (down + (u32)j)) : -1;
    }
    u32 avg[PARTS], root[PARTS], turn[PARTS];
    float as[PARTS], rs[PARTS], as2[PARTS], rs2[PARTS];
#pragma unroll
    for (int j = 0; j < PARTS; j++) {
        avg[j] = root[j] = 0;
        as[j] = rs[j] = as2[j] = rs2[j] = 0.0f;
        turn[j] = 4;
        if ((unsigned long long)source[j] >= (unsigned long long)t.src_rows) continue;
        const Place from = SINGLE ? (Place)source[j] : (Place)source[j] * (Place)cols + (j == 0 ? col : 0u), block = from >> 8;
        if (SINGLE) {
            avg[j] = t.src_avg[from];
            root[j] = t.src_root[from];
        } else {
            const u32 n = (j + 1 < PARTS && first[j + 1] < count ? first[j + 1] : count) - first[j];
            if (from + 4 <= (Place)(t.src_rows * t.cols)) {  // bytes behind the n are another row's, and dropped
                avg[j] = *reinterpret_cast<const u32_anywhere*>(t.src_avg + from);
                root[j] = *reinterpret_cast<const u32_anywhere*>(t.src_root + from);
            } else {
                for (u32 e = 0; e < n; e++) {
                    avg[j] |= (u32)t.src_avg[from + e] << (8 * e);
                    root[j] |= (u32)t.src_root[from + e] << (8 * e);
                }
            }
            const u32 left = 256u - ((u32)from & 255u);
            if (left < n) {
                turn[j] = first[j] + left;
                as2[j] = t.src_avg_scale[block + 1];
                rs2[j] = t.src_root_scale[block + 1];
            }
        }
        as[j] = t.src_avg_scale[block];
        rs[j] = t.src_root_scale[block];
    }
    u32 a = avg[0], r = root[0];
#pragma unroll
    for (int j = 1; j < PARTS; j++) {
        if (first[j] >= count) continue;  // first[j] is 1 to 3
        const u32 below = (1u << (8 * first[j])) - 1u;
        a = (a & below) | avg[j] << (8 * first[j]);
        r = (r & below) | root[j] << (8 * first[j]);
    }
    const u32 there = count ? ~0u >> (32 - 8 * count) : 0u;
    a &= there;
    r &= there;
    x[0] = __builtin_amdgcn_cvt_f32_fp8((int)a, 0) * as[0];
    y[0] = __builtin_amdgcn_cvt_f32_fp8((int)r, 0) * rs[0];
#pragma unroll
    for (u32 e = 1; e < 4; e++) {
        float sa = as[0], sr = rs[0];
#pragma unroll
        for (int j = 0; j < PARTS; j++) {
            if (j > 0 && (SINGLE ? e == (u32)j : e >= first[j])) sa = as[j], sr = rs[j];
            if (!SINGLE && e >= turn[j]) sa = as2[j], sr = rs2[j];
        }
        x[e] = (e == 1   ? __builtin_amdgcn_cvt_f32_fp8((int)a, 1)
                : e == 2 ? __builtin_amdgcn_cvt_f32_fp8((int)a, 2)
                         : __builtin_amdgcn_cvt_f32_fp8((int)a, 3)) * sa;
        y[e] = (e == 1   ? __builtin_amdgcn_cvt_f32_fp8((int)r, 1)
                : e == 2 ? __builtin_amdgcn_cvt_f32_fp8((int)r, 2)
                         : __builtin_amdgcn_cvt_f32_fp8((int)r, 3)) * sr;
    }
}

// The largest magnitude of four values, as its bits: their order is that of the magnitudes, and comparing
// them takes no quieting of NaNs.  What is not finite is left out, and told in `bad`.
__device__ __forceinline__ u32 top_bits(const float* x, bool& bad) {
    u32 bits[4];
#pragma unroll
    for (int e = 0; e < 4; e++) bits[e] = __float_as_uint(x[e]) & 0x7fffffffu;
    u32 top = max(max(bits[0], bits[1]), max(bits[2], bits[3]));
    bad = top >= 0x7f800000u;
    if (__builtin_expect(bad, 0)) {
        top = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) top = max(top, bits[e] < 0x7f800000u ? bits[e] : 0u);
    }
    return top;
}
__device__ __forceinline__ u32 wave_max_bits(u32 x) {
    x = max(x, (u32)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xf, 0xf, true));
    x = max(x, (u32)__builtin_amdgcn_mov_dpp((int)x, 0x124, 0xf, 0xf, true));
    x = max(x, (u32)__builtin_amdgcn_mov_dpp((int)x, 0x122, 0xf, 0xf, true));
    x = max(x, (u32)__builtin_amdgcn_mov_dpp((int)x, 0x121, 0xf, 0xf, true));
    x = max(x, (u32)__shfl_xor((int)x, 16, 64));
    return max(x, (u32)__shfl_xor((int)x, 32, 64));
}

// e4m3 codes of four values times inv, each the nearest, in their order from the lowest byte on; `bad`: one is not
// finite.  A square root above 0 has at least the least code, 2^-9.
__device__ __forceinline__ u32 encode_nearest4(const float* x, float inv, bool roots, bool bad) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; e++)
        y[e] = __builtin_amdgcn_fmed3f(x[e] * inv, !roots ? -448.0f : x[e] > 0.0f ? 0x1p-9f : 0.0f, 448.0f);
    u32 codes = (u32)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false), true);
    if (__builtin_expect(bad, 0)) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (!is_finite(x[e])) codes = (codes & ~(0xffu << (8 * e))) | (0x7fu | (__float_as_uint(x[e]) >> 31 << 7)) << (8 * e);
    }
    return codes;
}

// A wave's block of moments and square roots to codes and scales, each lane having four consecutive
// elements, `count` of which there are (the others are zero)
__device__ __forceinline__ void store_block(unsigned char* avg, unsigned char* root, float* avg_scale, float* root_scale,
                                            bool aligned, long long block, u32 count, const float* x, const float* y) {
    float minv, rinv, mscale, rscale;
    bool mbad, rbad;
    scales_of(__uint_as_float(wave_max_bits(top_bits(x, mbad))), mscale, minv);
    scales_of(__uint_as_float(wave_max_bits(top_bits(y, rbad))), rscale, rinv);
    const u32 c = encode_nearest4(x, minv, false, mbad), d = encode_nearest4(y, rinv, true, rbad);
    const long long begin = block * 256;
    if (aligned && count == 4) {
        reinterpret_cast<u32*>(avg + begin)[__lane_id()] = c;
        reinterpret_cast<u32*>(root + begin)[__lane_id()] = d;
    } else {
        for (u32 e = 0; e < count; e++) {
            avg[begin + 4 * __lane_id() + e] = (unsigned char)(c >> (8 * e));
            root[begin + 4 * __lane_id() + e] = (unsigned char)(d >> (8 * e));
        }
    }
    if (__lane_id() == 0) {
        avg_scale[block] = mscale;
        root_scale[block] = rscale;
    }
}

// An out block of 256 elements to a wave, four consecutive ones to a lane.  Divisions by cols
// are products: with (2^64 - 1) / cols + 1 once a wave (exact while the dividend times cols is below
// 2^64), and for what is left, below cols + 256, with ceil(2^20 / cols), or one comparison (cols >= 256).
// Bound by its instructions for the most part: 23.2M elements of rows of 1 to 4, 164 MB, take 41 us (a
// copy's rate would be 28) and 18.8M vector instructions, about 27 us of that: an addition, product, mask
// or move issues in 1.0 ns a SIMD here, a shift, select, comparison, maximum or conversion, six in ten of
// them, in 1.75.  Eight blocks a wave, one after another, 65 against 51 us then; two
// at once 57 against 55.
__global__ void __launch_bounds__(256) k_moment_rows(MomentRowsTable a) {
    const int k = find_tensor<MR_TENSORS>(a.first, a.count, blockIdx.x);
    const MomentRows t = a.t[k];
    const long long n = t.rows * t.cols;
    const u32 cols = (u32)t.cols;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // all of this is the wave's, in scalars
    const long long block = (long long)(blockIdx.x - a.first[k]) * 4 + wave, begin = block * 256;
    if (begin >= n) return;
    const long long row0 = t.reciprocal64 ? (long long)__umul64hi((unsigned long long)begin, t.reciprocal64) : begin;
    const u32 left = n - begin < 256 ? (u32)(n - begin) : 256u, i = 4 * __lane_id();
    const u32 count = i < left ? (left - i < 4 ? left - i : 4u) : 0u;
    const u32 at = (u32)(begin - row0 * t.cols) + i;
    const u32 down = cols < 256 ? (at * t.reciprocal) >> 20 : (at >= cols ? 1u : 0u);
    float x[4], y[4];
    const long long* index = t.index + row0;
    const u32 col = at - down * cols;
    if (t.src_rows * t.cols >= 1ll << 31)
        cols >= 3 ? gather<unsigned long long, 2>(t, index, down, col, count, x, y)
                  : gather<unsigned long long, 4>(t, index, down, col, count, x, y);
    else if ((cols & 3u) == 0)
        gather<u32, 1>(t, index, down, col, count, x, y);
    else if (cols >= 3)
        gather<u32, 2>(t, index, down, col, count, x, y);
    else if (cols == 2)
        gather<u32, 3>(t, index, down, col, count, x, y);
    else
        gather<u32, 4, true>(t, index, down, 0, count, x, y);
    store_block(t.avg, t.root, t.avg_scale, t.root_scale, t.aligned, block, count, x, y);
}

// How many of a lane's four elements of a block there are
__device__ __forceinline__ u32 lane_count(long long begin, long long n) {
    const long long left = n - begin - 4 * __lane_id();
    return left >= 4 ? 4u : left > 0 ? (u32)left : 0u;
}
__device__ __forceinline__ bool at_multiples(const void* p, const void* q, uintptr_t mask) {
    return ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & mask) == 0;
}

// 32-bit moments to codes, a wave a block.  23.3M elements, 233 MB: 39 us, decoded 37 (one element of a
// lane after another 68 and 51).
__global__ void __launch_bounds__(256) k_moments_encode(long long n, const float* __restrict__ exp_avg,
                                                        const float* __restrict__ exp_avg_sq, unsigned char* avg,
                                                        unsigned char* root, float* avg_scale, float* root_scale) {
    const long long block = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), begin = block * 256;
    if (begin >= n) return;
    const u32 count = lane_count(begin, n);
    float x[4], y[4];
    if (at_multiples(exp_avg, exp_avg_sq, 15u) && count == 4) {
        const float4 m = load_once(reinterpret_cast<const float4*>(exp_avg + begin) + __lane_id());
        const float4 v = load_once(reinterpret_cast<const float4*>(exp_avg_sq + begin) + __lane_id());
        x[0] = m.x, x[1] = m.y, x[2] = m.z, x[3] = m.w;
        y[0] = v.x, y[1] = v.y, y[2] = v.z, y[3] = v.w;
    } else {
#pragma unroll
        for (u32 e = 0; e < 4; e++) {
            x[e] = e < count ? exp_avg[begin + 4 * __lane_id() + e] : 0.0f;
            y[e] = e < count ? exp_avg_sq[begin + 4 * __lane_id() + e] : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = sqrtf(y[e]);
    store_block(avg, root, avg_scale, root_scale, at_multiples(avg, root, 3u), block, count, x, y);
}

__global__ void __launch_bounds__(256) k_moments_decode(long long n, const unsigned char* __restrict__ avg,
                                                        const unsigned char* __restrict__ root,
                                                        const float* __restrict__ avg_scale,
                                                        const float* __restrict__ root_scale, float* exp_avg,
                                                        float* exp_avg_sq) {
    const long long block = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), begin = block * 256;
    if (begin >= n) return;
    const u32 count = lane_count(begin, n);
    const float as = avg_scale[block], rs = root_scale[block];
    if (at_multiples(avg, root, 3u) && at_multiples(exp_avg, exp_avg_sq, 15u) && count == 4) {
        const u32 c = load_once(reinterpret_cast<const u32*>(avg + begin) + __lane_id());
        const u32 d = load_once(reinterpret_cast<const u32*>(root + begin) + __lane_id());
        reinterpret_cast<float4*>(exp_avg + begin)[__lane_id()] =
            make_float4(decode(c) * as, decode(c >> 8) * as, decode(c >> 16) * as, decode(c >> 24) * as);
        reinterpret_cast<float4*>(exp_avg_sq + begin)[__lane_id()] =
            make_float4(square(decode(d) * rs), square(decode(d >> 8) * rs), square(decode(d >> 16) * rs), square(decode(d >> 24) * rs));
    } else {
        for (u32 e = 0; e < count; e++) {
            const long long i = begin + 4 * __lane_id() + e;
            exp_avg[i] = decode(avg[i]) * as;
            exp_avg_sq[i] = square(decode(root[i]) * rs);
        }
    }
}

// ---- the global norm ----------------------------------------------------------------------

// Bound by HBM: 1 GB at 5.8, 4 GB at 6.2 TB/s, launches and the joining of the partials included.

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
}

__device__ __forceinline__ double square64(float x) { return (double)x * (double)x; }

// Four waves' sums, in their order, in thread 0
__device__ __forceinline__ double group_sum(double x, double* sh) {
    x = wave_sum(x);
    if (__lane_id() == 0) sh[threadIdx.x >> 6] = x;
    __syncthreads();
    return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// A workgroup's part of its tensor
struct NormPart {
    void* g;
    long long lo, hi;
    int type;
    bool aligned;  // g begins at a multiple of four elements
};
__device__ __forceinline__ NormPart norm_part(const NormTable& a) {
    const int k = find_tensor<NORM_TENSORS>(a.first, a.count, blockIdx.x);
    const NormTensor t = a.t[k];
    const u32 end = k + 1 < a.count ? a.first[k + 1] : gridDim.x;
    NormPart p;
    p.g = reinterpret_cast<void*>((uintptr_t)t.g);
    p.type = (int)t.type;
    p.aligned = ((u32)t.g & (p.type == AW_F32 ? 15u : 7u)) == 0;
    p.lo = (long long)(blockIdx.x - a.first[k]) * NORM_CHUNK;
    p.hi = p.lo + (blockIdx.x + 1 == end ? (int)t.tail : NORM_CHUNK);
    return p;
}

// The sum of squares of a workgroup's elements of type T; whole rounds of NORM_ROUND elements are
// vectors, the next round's loads in flight while one is summed
template <int T>
__device__ __forceinline__ double chunk_squares(const NormPart& t) {
    double sum = 0.0;
    long long lo = t.lo;
    const long long hi = t.hi;
    if (t.aligned) {
        constexpr int V = NORM_ROUND / 1024;
        const typename Vec4<T>::raw* g = vec4<T>(t.g) + (lo >> 2) + threadIdx.x;
        typename Vec4<T>::raw x[V], next[V];
        long long rounds = (hi - lo) / NORM_ROUND;
        lo += rounds * NORM_ROUND;
        if (rounds) {
#pragma unroll
            for (int j = 0; j < V; j++) x[j] = g[256 * j];
        }
        while (rounds--) {
            g += 256 * V;
            if (rounds) {
#pragma unroll
                for (int j = 0; j < V; j++) next[j] = g[256 * j];
            }
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float4 y = Vec4<T>::get(x[j]);
                sum += (square64(y.x) + square64(y.y)) + (square64(y.z) + square64(y.w));
                x[j] = next[j];
            }
        }
    }
    for (long long i = lo + threadIdx.x; i < hi; i += 256) sum += square64(load_as_float(t.g, T, i));
    return sum;
}

// Sums of squares in 64 bits: no overflow of g g, and each partial in a fixed order
__global__ void __launch_bounds__(256) k_norm_partial(NormTable a, double* __restrict__ partial) {
    __shared__ double sh[4];
    const NormPart t = norm_part(a);
    double sum;
    if (t.type == AW_F32)
        sum = chunk_squares<AW_F32>(t);
    else if (t.type == AW_BF16)
        sum = chunk_squares<AW_BF16>(t);
    else
        sum = chunk_squares<AW_F16>(t);
    sum = group_sum(sum, sh);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// Many partials: each workgroup joins 4096 of them in place of its first
__global__ void __launch_bounds__(256) k_norm_join(const double* __restrict__ partial, long long n,
                                                   double* __restrict__ joined) {
    __shared__ double sh[4];
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const long long i = (long long)blockIdx.x * 4096 + 256 * j + threadIdx.x;
        if (i < n) sum += partial[i];
    }
    sum = group_sum(sum, sh);
    if (threadIdx.x == 0) joined[blockIdx.x] = sum;
}

// out = (norm, min(1, max_norm / (norm + 1e-6))), norm = scale sqrt(sum); one workgroup, whose
// threads have 16 partials each in flight
__global__ void __launch_bounds__(256) k_norm_final(const double* __restrict__ partial, long long n, double scale,
                                                    double max_norm, float* out) {
    __shared__ double sh[4];
    double sum = 0.0;
    for (long long at = 0; at < n; at += 4096) {
        double x[16];
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const long long i = at + 256 * j + threadIdx.x;
            x[j] = i < n ? partial[i] : 0.0;
        }
#pragma unroll
        for (int j = 0; j < 16; j++) sum += x[j];
    }
    sum = group_sum(sum, sh);
    if (threadIdx.x == 0) {
        const double norm = scale * sqrt(sum);
        const double coef = max_norm / (norm + 1e-6);
        out[0] = (float)norm;
        out[1] = (float)(coef > 1.0 ? 1.0 : coef);  // NaN stays NaN
    }
}

// The same sums over a step's tensors, a wave to each of their groups of G elements: what a step
// reads anyway finds its gradients, and a list in memory is looked up by one launch.
template <int T, int G>
__device__ __forceinline__ double group_squares(const AdamWTensor& t, long long lo, long long hi) {
    double sum = 0.0;
    if (t.aligned && hi - lo == G) {
        const typename Vec4<T>::raw* g = vec4<T>(t.g) + (lo >> 2) + __lane_id();
        typename Vec4<T>::raw x[G / 256];
#pragma unroll
        for (int j = 0; j < G / 256; j++) x[j] = g[64 * j];
#pragma unroll
        for (int j = 0; j < G / 256; j++) {
            const float4 y = Vec4<T>::get(x[j]);
            sum += (square64(y.x) + square64(y.y)) + (square64(y.z) + square64(y.w));
        }
    } else {
        for (long long i = lo + __lane_id(); i < hi; i += 64) sum += square64(load_as_float(t.g, T, i));
    }
    return sum;
}

template <int G>
__device__ __forceinline__ double squares_of(const AdamWTensor& t, u32 group) {
    const long long lo = (long long)group * G, hi = lo + G < t.n ? lo + G : t.n;
    if (t.grad_type == AW_F32) return group_squares<AW_F32, G>(t, lo, hi);
    if (t.grad_type == AW_BF16) return group_squares<AW_BF16, G>(t, lo, hi);
    return group_squares<AW_F16, G>(t, lo, hi);
}

// Four groups a workgroup, the last ones first: 77.4M fp32 gradients between two steps 81 us, from the
// first 95 (the step takes as long after either).  With loads past the caches 47 us, but the last step's stores
// are then written out during this one: 230 us, and 63.5M bf16 ones 37 + 322 against 53 + 261 us.
template <int U>
__global__ void __launch_bounds__(256) k_adamw_squares(AdamWTable a, u32 groups, double* __restrict__ partial) {
    __shared__ double sh[4];
    const u32 group = __builtin_amdgcn_readfirstlane(groups - 1 - (blockIdx.x * 4 + (threadIdx.x >> 6)));  // wraps: none
    double sum = 0.0;
    if (group < groups) {
        const int k = find_tensor<AW_TENSORS>(a.first, a.count, group);
        const AdamWTensor t = a.t[k];
        sum = squares_of<1024 * U>(t, group - a.first[k]);
    }
    sum = group_sum(sum, sh);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

template <int U>
__global__ void __launch_bounds__(256) k_adamw_squares_many(int count, const u32* __restrict__ first,
                                                            const AdamWTensor* __restrict__ list, u32 groups,
                                                            double* __restrict__ partial) {
    __shared__ double sh[4];
    const u32 group = __builtin_amdgcn_readfirstlane(groups - 1 - (blockIdx.x * 4 + (threadIdx.x >> 6)));  // wraps: none
    double sum = 0.0;
    if (group < groups) {
        const int k = find_tensor_in(first, count, group);
        const AdamWTensor t = list[k];
        sum = squares_of<1024 * U>(t, group - first[k]);
    }
    sum = group_sum(sum, sh);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

template <int T>
__device__ __forceinline__ void chunk_scale(const NormPart& t, float coef) {
    const long long lo = t.lo, hi = t.hi;
    if (t.aligned && hi - lo == NORM_CHUNK) {
        constexpr int V = NORM_CHUNK / 1024;
        typename Vec4<T>::raw* g = vec4<T>(t.g) + (lo >> 2) + threadIdx.x;
        typename Vec4<T>::raw x[V];
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = g[256 * j];
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float4 y = Vec4<T>::get(x[j]);
            g[256 * j] = Vec4<T>::put(make_float4(y.x * coef, y.y * coef, y.z * coef, y.w * coef));
        }
    } else {
        for (long long i = lo + threadIdx.x; i < hi; i += 256)
            store_from_float(t.g, T, i, load_as_float(t.g, T, i) * coef);
    }
}

__global__ void __launch_bounds__(256) k_grad_scale(NormTable a, const float* __restrict__ clip) {
    const NormPart t = norm_part(a);
    const float coef = clip[1];
    if (t.type == AW_F32)
        chunk_scale<AW_F32>(t, coef);
    else if (t.type == AW_BF16)
        chunk_scale<AW_BF16>(t, coef);
    else
        chunk_scale<AW_F16>(t, coef);
}

}  // namespace

void launch_adamw(const AdamWTable& a, unsigned grid, int bits, int u, hipStream_t st) {
    if (bits == 8 && u == 2)
        hipLaunchKernelGGL((k_adamw<8, 2>), dim3(grid), dim3(256), 0, st, a);
    else if (bits == 8)
        hipLaunchKernelGGL((k_adamw<8, 1>), dim3(grid), dim3(256), 0, st, a);
    else if (u == 2)
        hipLaunchKernelGGL((k_adamw<32, 2>), dim3(grid), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((k_adamw<32, 1>), dim3(grid), dim3(256), 0, st, a);
}

void launch_adamw_list(const AdamWTable& a, unsigned* first, AdamWTensor* list, hipStream_t st) {
    hipLaunchKernelGGL(k_adamw_list, dim3(1), dim3(256), 0, st, a, first, list);
}

void launch_adamw_many(const AdamWCall& a, const AdamWRates& rates, int count, const unsigned* first,
                       const AdamWTensor* list, unsigned grid, int bits, int u, hipStream_t st) {
    if (bits == 8 && u == 2)
        hipLaunchKernelGGL((k_adamw_many<8, 2>), dim3(grid), dim3(256), 0, st, a, rates, count, first, list);
    else if (bits == 8)
        hipLaunchKernelGGL((k_adamw_many<8, 1>), dim3(grid), dim3(256), 0, st, a, rates, count, first, list);
    else if (u == 2)
        hipLaunchKernelGGL((k_adamw_many<32, 2>), dim3(grid), dim3(256), 0, st, a, rates, count, first, list);
    else
        hipLaunchKernelGGL((k_adamw_many<32, 1>), dim3(grid), dim3(256), 0, st, a, rates, count, first, list);
}

void launch_adamw_squares(const AdamWTable& a, unsigned groups, double* partial, int u, hipStream_t st) {
    const dim3 grid((groups + 3) / 4);
    if (u == 2)
        hipLaunchKernelGGL(k_adamw_squares<2>, grid, dim3(256), 0, st, a, groups, partial);
    else
        hipLaunchKernelGGL(k_adamw_squares<1>, grid, dim3(256), 0, st, a, groups, partial);
}

void launch_adamw_squares_many(int count, const unsigned* first, const AdamWTensor* list, unsigned groups,
                               double* partial, int u, hipStream_t st) {
    const dim3 grid((groups + 3) / 4);
    if (u == 2)
        hipLaunchKernelGGL(k_adamw_squares_many<2>, grid, dim3(256), 0, st, count, first, list, groups, partial);
    else
        hipLaunchKernelGGL(k_adamw_squares_many<1>, grid, dim3(256), 0, st, count, first, list, groups, partial);
}

void launch_adamw_scalars(const AdamWCounts& a, hipStream_t st) {
    hipLaunchKernelGGL(k_adamw_scalars, dim3(1), dim3(64), 0, st, a);
}

void launch_moment_rows(const MomentRowsTable& a, unsigned grid, hipStream_t st) {
    hipLaunchKernelGGL(k_moment_rows, dim3(grid), dim3(256), 0, st, a);
}

void launch_moments_encode(long long n, const float* exp_avg, const float* exp_avg_sq, unsigned char* avg,
                           unsigned char* root, float* avg_scale, float* root_scale, hipStream_t st) {
    hipLaunchKernelGGL(k_moments_encode, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, st, n, exp_avg, exp_avg_sq,
                       avg, root, avg_scale, root_scale);
}

void launch_moments_decode(long long n, const unsigned char* avg, const unsigned char* root, const float* avg_scale,
                           const float* root_scale, float* exp_avg, float* exp_avg_sq, hipStream_t st) {
    hipLaunchKernelGGL(k_moments_decode, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, st, n, avg, root, avg_scale,
                       root_scale, exp_avg, exp_avg_sq);
}

void launch_norm_partial(const NormTable& a, unsigned grid, double* partial, hipStream_t st) {
    hipLaunchKernelGGL(k_norm_partial, dim3(grid), dim3(256), 0, st, a, partial);
}

void launch_norm_join(const double* partial, long long n, double* joined, hipStream_t st) {
    hipLaunchKernelGGL(k_norm_join, dim3((unsigned)((n + 4095) / 4096)), dim3(256), 0, st, partial, n, joined);
}

void launch_norm_final(const double* partial, long long n, double scale, double max_norm, float* out, hipStream_t st) {
    hipLaunchKernelGGL(k_norm_final, dim3(1), dim3(256), 0, st, partial, n, scale, max_norm, out);
}

void launch_grad_scale(const NormTable& a, unsigned grid, const float* clip, hipStream_t st) {
    hipLaunchKernelGGL(k_grad_scale, dim3(grid), dim3(256), 0, st, a, clip);
}

}  // namespace gsr
