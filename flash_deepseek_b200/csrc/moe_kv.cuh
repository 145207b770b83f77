// moe_kv.cuh -- the paged latent cache of MLA attention as the kernels see
// it: row formats, the page table, the rows of a batch's sequences.
//
// A cache row is L latent values and MOE_KV_ROPE rotary values.  16-bit
// formats: L + 64 values one after the other.  8-bit formats: L e4m3 codes,
// 64 rotary values of 16 bits, L / 32 scale bytes (127 + k: the 32 codes of a
// group stand for code * 2^k), padded to 16 bytes.  A power-of-two scale makes
// every stored value exact in fp16 and bf16 (k is kept in [-15, 7]: e4m3 spans
// 2^-9 .. 448, so code * 2^k stays within fp16's 2^-24 .. 65504), so the
// attention kernel's 16-bit operands hold exactly what the cache holds.
// Scale byte 255: the group held an infinity or a NaN and reads as NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "../../include/moe_cuda.h"
#include "moe_internal.h"

#define KV_GROUP 32
#define KV_K_MIN (-15)
#define KV_K_MAX 7

__device__ __forceinline__ void kv_error(int *error, int code) { atomicExch(error, code); }

// The sequence that row t of the batch belongs to (the last b with
// q_start[b] <= t < q_start[b + 1]), or -1: rows in front of the first
// sequence and behind the last one belong to none.
__device__ __forceinline__ int kv_seq_of(const MoeKvBatchDev &b, int t) {
    int lo = 0, hi = b.n_seqs + 1;   // first index whose start is above t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(b.q_start + mid) <= t) lo = mid + 1;
        else hi = mid;
    }
    return lo == 0 || lo > b.n_seqs ? -1 : lo - 1;
}

// Row `pos` of sequence `seq` in the cache as a flat row number, or -1 when
// the page table does not hold it (position or page out of range).
__device__ __forceinline__ long long kv_flat_row(const MoeKvDev &kv, const MoeKvBatchDev &b, int seq, long long pos) {
    const long long pi = pos >> kv.page_shift;
    if (pos < 0 || pi >= b.pages_per_seq) return -1;
    const int page = __ldg(b.pages + (size_t)seq * b.pages_per_seq + pi);
    if (page < 0 || page >= kv.n_pages) return -1;
    return ((long long)page << kv.page_shift) + (pos & ((1 << kv.page_shift) - 1));
}

// ---- element types ---------------------------------------------------------
template <typename T> struct KvType;
template <> struct KvType<float> {
    static __device__ __forceinline__ float to_f(float v) { return v; }
    static __device__ __forceinline__ float from_f(float v) { return v; }
};
template <> struct KvType<__half> {
    static __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
};
template <> struct KvType<__nv_bfloat16> {
    static __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
};

// 8 consecutive values; VEC: 16-byte aligned, whole-vector accesses
template <typename T, bool VEC>
__device__ __forceinline__ void kv_load8(const T *p, float (&v)[8]) {
    T t[8];
    if (VEC) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) * 8 / 16); i++)
            reinterpret_cast<uint4 *>(t)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) t[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = KvType<T>::to_f(t[i]);
}
template <typename T, bool VEC>
__device__ __forceinline__ void kv_store8(T *p, const float (&v)[8]) {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = KvType<T>::from_f(v[i]);
    if (VEC) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) * 8 / 16); i++)
            reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(t)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = t[i];
    }
}

// the same 8 values as loaded (2 or 1 registers a pair instead of 2): what a
// thread holds of loads that are under way
template <typename T> struct KvRaw8 { uint4 q[sizeof(T) / 2]; };
// (RW: memory that the kernel itself writes, so not through the read-only path, which is faster: 86 against 100 us for
// 4096 tokens x 128 heads x 192 rotated)
template <typename T, bool RW = false>
__device__ __forceinline__ void kv_load_raw(const T *p, KvRaw8<T> &r) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); i++) r.q[i] = RW ? reinterpret_cast<const uint4 *>(p)[i] : __ldg(reinterpret_cast<const uint4 *>(p) + i);
}
template <typename T>
__device__ __forceinline__ void kv_unraw(const KvRaw8<T> &r, float (&v)[8]) {
    const T *t = reinterpret_cast<const T *>(r.q);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = KvType<T>::to_f(t[i]);
}

// 4 e4m3 codes (a 32-bit word) to fp32; exact
__device__ __forceinline__ void kv_e4m3x4(uint32_t w, float *v) {
    const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFF), __NV_E4M3);
    const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
    const float2 fa = __half22float2(__half2(a)), fb = __half22float2(__half2(b));
    v[0] = fa.x, v[1] = fa.y, v[2] = fb.x, v[3] = fb.y;
}

// cos and sin of pos * freq, freq given as turns per position.  The product
// and its reduction to half a turn run in 64 bits (an fp32 product at
// position 10^5 is off by 10^-3 radians); the reduced angle, at most half a
// turn, keeps fp32's relative precision.
__device__ __forceinline__ void kv_cos_sin(int pos, double turns_per_pos, float mscale, float &c, float &s) {
    const double turns = (double)pos * turns_per_pos;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    c *= mscale;
    s *= mscale;
}
