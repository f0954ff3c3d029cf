// Pairs of 32-bit values that one instruction takes together, each rounded as by itself.
#pragma once

namespace b2 {

struct Two { unsigned long long v; };
__device__ __forceinline__ Two two(float a, float b) { Two r; asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ Two two(float a) { return two(a, a); }
__device__ __forceinline__ float2 apart(Two a) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v)); return r; }
__device__ __forceinline__ Two operator*(Two a, Two b) { Two r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ Two operator+(Two a, Two b) { Two r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) { Two r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }

}  // namespace b2
