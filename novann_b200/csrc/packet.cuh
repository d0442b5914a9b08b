// Vectors of fp32 / fp16 / bf16 elements: loads widened to fp32, stores rounded to nearest even.
#pragma once

#include "nvq_common.cuh"

#ifdef __CUDACC__
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float f16_bits_to_f32(uint32_t h) {
    float f;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.f32.f16 %0, t;\n\t}" : "=f"(f) : "r"(h));
    return f;
}

// Element type DT (an nvq_dtype): its storage word and the conversions of one 32-bit word of it.
template <int DT> struct Elem;
template <> struct Elem<NVQ_F32> {
    using type = float;
    static constexpr int SIZE = 4, PER_WORD = 1;
    static __device__ __forceinline__ void widen(uint32_t w, float* f) { f[0] = __uint_as_float(w); }
    static __device__ __forceinline__ uint32_t narrow(const float* f) { return __float_as_uint(f[0]); }
    static __device__ __forceinline__ float load(const void* p) { return *(const float*)p; }
    static __device__ __forceinline__ void store(void* p, float v) { *(float*)p = v; }
};
template <> struct Elem<NVQ_F16> {
    using type = uint16_t;
    static constexpr int SIZE = 2, PER_WORD = 2;
    static __device__ __forceinline__ void widen(uint32_t w, float* f) {
        f[0] = f16_bits_to_f32(w & 0xFFFFu);
        f[1] = f16_bits_to_f32(w >> 16);
    }
    static __device__ __forceinline__ uint32_t narrow(const float* f) { return pack_f16x2(f[0], f[1]); }
    static __device__ __forceinline__ float load(const void* p) { return f16_bits_to_f32(*(const uint16_t*)p); }
    static __device__ __forceinline__ void store(void* p, float v) { *(uint16_t*)p = (uint16_t)pack_f16x2(v, v); }
};
template <> struct Elem<NVQ_BF16> {
    using type = uint16_t;
    static constexpr int SIZE = 2, PER_WORD = 2;
    static __device__ __forceinline__ void widen(uint32_t w, float* f) {
        f[0] = __uint_as_float(w << 16);
        f[1] = __uint_as_float(w & 0xFFFF0000u);
    }
    static __device__ __forceinline__ uint32_t narrow(const float* f) { return pack_bf16x2(f[0], f[1]); }
    static __device__ __forceinline__ float load(const void* p) {
        return __uint_as_float((uint32_t)*(const uint16_t*)p << 16);
    }
    static __device__ __forceinline__ void store(void* p, float v) { *(uint16_t*)p = (uint16_t)pack_bf16x2(v, v); }
};

// V consecutive elements at p (aligned to their own size together) as raw words, and their widening
template <int DT, int V> struct Packet {
    using E = Elem<DT>;
    static constexpr int BYTES = V * E::SIZE;
    static constexpr int WORDS = BYTES >= 4 ? BYTES / 4 : 1;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const void* p) {
        if constexpr (BYTES == 16) {
            const uint4 r = *(const uint4*)p;
            w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
        } else if constexpr (BYTES == 4) {
            w[0] = *(const uint32_t*)p;
        } else {
            static_assert(BYTES == 2, "packets are 16, 4 or 2 bytes");
            w[0] = *(const uint16_t*)p;
        }
    }
    // read once: not kept in L1
    __device__ __forceinline__ void load_stream(const void* p) {
        if constexpr (BYTES == 16) {
            const uint4 r = ldg_stream_128(p);
            w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w;
        } else {
            load(p);
        }
    }
    // the same for memory that this kernel may write (in place)
    __device__ __forceinline__ void load_once(const void* p) {
        if constexpr (BYTES == 16) {
            asm volatile("ld.global.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "l"(p)
                         : "memory");
        } else {
            load(p);
        }
    }
    __device__ __forceinline__ void store(void* p) const {
        if constexpr (BYTES == 16) stg_stream_128(p, make_uint4(w[0], w[1], w[2], w[3]));
        else if constexpr (BYTES == 4) *(uint32_t*)p = w[0];
        else *(uint16_t*)p = (uint16_t)w[0];
    }
    __device__ __forceinline__ void widen(float* f) const {
        if constexpr (BYTES == 2) {
            float t[2];
            E::widen(w[0], t);
            f[0] = t[0];
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i++) E::widen(w[i], f + i * E::PER_WORD);
        }
    }
    __device__ __forceinline__ void narrow(const float* f) {
        if constexpr (BYTES == 2) {
            const float t[2] = {f[0], f[0]};
            w[0] = E::narrow(t);
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i++) w[i] = E::narrow(f + i * E::PER_WORD);
        }
    }
};
#endif
