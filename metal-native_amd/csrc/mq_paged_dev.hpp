// Device-side building blocks of the paged-cache kernels (gfx950 only).
#pragma once
#include "mq_paged.hpp"
#include "mq_device.hpp"

namespace mq {
namespace {

typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

struct F16 {
  typedef _Float16 e;
  static constexpr uint32_t kExp = 0x7C007C00u, kExpLow = 0x04000400u;   // exponent fields of two values, their lowest bits
  static __device__ __forceinline__ f16v mfma(u4 a, u4 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
  // c += a b in c's own registers: from the builtin the result goes to others
  // wherever c also lives on another path.  The compiler does not see the
  // latency: operands that a vector instruction writes are written two
  // instructions before, and c is not touched but by such products for 20.
  static __device__ __forceinline__ void add(f16v& c, u4 a, u4 b) {
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  }
};
struct BF16 {
  typedef __bf16 e;
  static constexpr uint32_t kExp = 0x7F807F80u, kExpLow = 0x00800080u;
  static __device__ __forceinline__ f16v mfma(u4 a, u4 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  }
  // c += a b in c's own registers: from the builtin the result goes to others
  // wherever c also lives on another path.  The compiler does not see the
  // latency: operands that a vector instruction writes are written two
  // instructions before, and c is not touched but by such products for 20.
  static __device__ __forceinline__ void add(f16v& c, u4 a, u4 b) {
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  }
};
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef typename T::e e2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){a, b}, e2));
}

// s <- softcap * tanh(scale * s / softcap) at any cap.  far: tanh y = 1 - 2 /
// (e^2y + 1) is off by about 5 e of the cap (e = 2^-24) whatever y is, which a
// cap far above the scores makes large; near: the series, off by 1 e of itself up
// to |y| = 1/4 (its next term is 9e-9) and half the instructions.  A wave none of
// whose scores is larger takes the series alone.  Otherwise, where a lane's scores
// are one row's (ONE_ROW), it takes far unless they all are under cap / 16: an
// error of the cap is one of that row's largest score then.  Else each score of
// its own size, but for caps whose error is no more than that of a sum of weights.
// Seven prompts, 28 heads over 4, 128 wide, bf16, cap 30 / 2 with scores N(0, 1):
// 121 / 128 us; each score by its size 123 / 189; far alone 122 / 121.
constexpr float kSmallCap = 32.f;
template <bool ONE_ROW, int N> __device__ __forceinline__ void cap_scores(f16v (&s)[N], const PagedArgs& p) {
  const float scale = p.scale, cap = p.softcap, inv = p.inv_cap, limit = 0.25f * cap;
  float top = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      s[n][j] *= scale;
      top = fmaxf(top, fabsf(s[n][j]));
    }
  auto near = [&](float x) {
    const float y = x * inv, z = y * y;
    float t = __builtin_fmaf(z, 62.f / 2835, -17.f / 315);
    t = __builtin_fmaf(z, t, 2.f / 15);
    t = __builtin_fmaf(z, t, -1.f / 3);
    return __builtin_fmaf(x * z, t, x);
  };
  auto far = [&](float x) {
    const float e = __builtin_amdgcn_exp2f(x * inv * (2.f * kLog2e));
    return cap * __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f);
  };
  auto each = [&](auto&& f) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int j = 0; j < 16; ++j) s[n][j] = f(s[n][j]);
  };
  if (!__any(top > limit)) {
    each(near);
  } else if (ONE_ROW) {
    if (top < 0.25f * limit) each(near);
    else each(far);
  } else if (cap <= kSmallCap) {
    each(far);
  } else {
    each([&](float x) {
      const float a = near(x), b = far(x);
      return fabsf(x) > limit ? b : a;
    });
  }
}

__device__ __forceinline__ float swap32(float v) {   // v of lane ^ 32
  const int x = __float_as_int(v);
  const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return __int_as_float((threadIdx.x & 32) ? (int)r[0] : (int)r[1]);
}
__device__ __forceinline__ int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ PagedSeq load_seq(const PagedArgs& p, int s) {
  return paged_seq(s, p.cu ? p.cu[s] : 0, p.cu ? p.cu[s + 1] : 0, p.cu != nullptr, p.lens[s],
                   p.prefix ? p.prefix[s] : 0, p.rows, p.cap);
}
__device__ __forceinline__ int64_t wave_scan(int64_t v) {   // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t t = __shfl_up(v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// Where a cache's slots lie for one key/value head, and the lane's part of a
// 1024-byte load: LDS is written in lane order, rows of D elements one after
// the other, and the 16-byte pieces of a row are permuted on their way (piece
// c of slot j at c ^ swizzle(j)) so that the reads below meet no bank twice.
template <int D> struct Lay {
  static constexpr int ROW = D / 8;           // 16-byte pieces of a slot
  static constexpr int GS = 64 / ROW;         // slots per load: 4 (D = 128) or 8 (64)
  static __device__ __forceinline__ int swz_k(int j) { return D == 128 ? j & 15 : (j >> 1) & 7; }
  // four pieces (32 lanes' 8 bytes) of four slots at a time
  static __device__ __forceinline__ int swz_v(int j) { return D == 128 ? 4 * (j & 3) : 4 * ((j >> 1) & 1); }
};

#if defined(__HIP_DEVICE_COMPILE__)
// 64 lanes' 16 bytes each at base + voff (zeros where voff + 16 > bytes) into
// 1024 bytes of LDS in lane order; base, bytes and lds are wave-uniform.  In
// asm, without an output: the builtin's load counts as a write that any later
// LDS read may depend on, and the compiler waits for the next tile's loads
// before it reads this tile.  Whoever reads the LDS waits for vmcnt itself;
// the compiler's own vmcnt waits only become stricter by loads it does not
// know of.  s_nop: M0, and a descriptor that v_readlane wrote (FRESH), need
// one and up to five wait states before the load.
typedef uint32_t desc_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ desc_t make_desc(const void* base, uint32_t bytes) {
  const uint64_t a = (uint64_t)base;
  return (desc_t){(uint32_t)uni((int)a), (uint32_t)uni((int)(a >> 32)) & 0xffffu, (uint32_t)uni((int)bytes), 0x00020000u};
}
template <bool FRESH> __device__ __forceinline__ void lds_load16(desc_t r, uint32_t voff, void* lds) {
  const uint32_t l = (uint32_t)uni((int)(uintptr_t)(__attribute__((address_space(3))) void*)lds);
  if constexpr (FRESH)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(l), "v"(voff), "s"(r) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(l), "v"(voff), "s"(r) : "memory");
}
__device__ __forceinline__ void lds_load16(const void* base, uint32_t bytes, uint32_t voff, void* lds) {
  lds_load16<true>(make_desc(base, bytes), voff, lds);
}
#else
typedef uint32_t desc_t __attribute__((ext_vector_type(4)));
__device__ inline desc_t make_desc(const void*, uint32_t) { return {}; }
template <bool FRESH> __device__ inline void lds_load16(desc_t, uint32_t, void*) {}
__device__ inline void lds_load16(const void*, uint32_t, uint32_t, void*) {}
#endif

struct Base {   // wave-uniform
  const char* ptr;      // of the key/value head
  uint32_t page, slot;  // bytes: below 2^32 each, and a page's slots together
  __device__ __forceinline__ const char* at(uint32_t id, uint32_t in_page) const {
    return ptr + ((uint64_t)id * page + in_page * slot);
  }
};
__device__ __forceinline__ Base cache_base(const PagedCache& c, int kv) {
  return {(const char*)c.ptr + 2 * kv * c.head, 2u * (uint32_t)c.page, 2u * (uint32_t)c.slot};
}

}  // namespace
}  // namespace mq
