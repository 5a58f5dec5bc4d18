// y = x W^T + bias for a few rows of x, W [N, K] in 4 bits: W[n, k] = (c[n, k] - z[n, k / g]) s[n, k / g], codes c and
// zeros z in 0 .. 15 (z = 8 where there are none), s in bf16, groups of g = 32, 64 or 128 columns.
//
// Bound by the bytes of the codes, which each wave streams as whole kilobytes: 16 features by 128 columns, laid out
// once as the MFMA wants them (shuffle4 below), a lane's 16 bytes the codes of its feature for four MFMAs. Codes become
// bf16 without arithmetic: 0x4300 | c is 128 + c exactly, so a pair of them costs an AND-OR and a shift. What that adds to a
// group's sum is taken off by a second MFMA whose weights are all -(128 + z), exact as well:
//
//   sum_k (128 + c) x  +  sum_k -(128 + z) x  =  sum_k (c - z) x,
//
// and the group's scale enters in f32. Products of whole numbers up to 143 with bf16 are exact, and what f32 sums lose, 2^-24
// of terms up to 143 |x| where the result's own are up to 15 |x|, is far below the result's rounding to bf16.
// (With sums of x from an MFMA of ones and the subtraction in f32, vector instructions bounded small groups: 28672 x 4096 for
// eight rows in groups of 64 with zeros 20 us; 17 to 19 by that clock, launches in a replayed graph, 14.3 among other calls.)
#include "common.h"

#define L4_TILE 16                     // features of a tile
#define L4_K 128                       // columns of a kilobyte

typedef unsigned l4_u4 __attribute__((ext_vector_type(4)));

// Codes as they come, two a byte, the lower half first: [N, K / 2]; -> [tile][K block][lane][4]: dword s of lane (feature
// li, fq) has columns 32 s + 8 fq + e of the block, e = 2 p in half-byte p, e = 2 p + 1 in half-byte p + 4. Zeros past N and K.
__global__ __launch_bounds__(256) void shuffle4_kernel(const unsigned char* src, unsigned* dst, int N, int K, int blocks, long long total) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int s = id & 3, lane = (id >> 2) & 63;
  const long long tb = id >> 8;
  const int kb = (int)(tb % blocks), n = (int)(tb / blocks) * L4_TILE + (lane & 15), k = kb * L4_K + 32 * s + 8 * (lane >> 4);
  unsigned w = 0;
  if (n < N && k < K) {                           // K is a multiple of 32
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const unsigned two = src[(size_t)n * (K / 2) + k / 2 + p];
      w |= (two & 15) << (4 * p) | (two >> 4) << (4 * p + 16);
    }
  }
  dst[id] = w;
}

// Scales [N, groups] -> [tile][K block][fq][group of the block][4]: a lane's four features (4 fq ..) of all groups side by side;
// zeros -> [tile][K block][feature][group of the block] as -(128 + z)'s lower byte, z. Zeros past N and K.
template <typename T, bool QUADS> __global__ __launch_bounds__(256) void shuffle4_groups_kernel(const T* src, T* dst, int N, int groups, int per,
                                                                                               int blocks, long long total) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int in = (int)(id % (16 * per));
  const long long tb = id / (16 * per);
  const int f = QUADS ? in / (4 * per) * 4 + in % 4 : in / per, g = (int)(tb % blocks) * per + (QUADS ? in / 4 % per : in % per);
  const long long n = tb / blocks * L4_TILE + f;
  dst[id] = n < N && g < groups ? src[n * groups + g] : (T)0;
}

extern "C" int loqa_shuffle4(const void* codes, const void* scales, const void* zeros, void* dst, void* dst_scales, void* dst_zeros, int N, int K,
                             int group, hipStream_t st) {
  if (N <= 0 || K <= 0 || K % 32 || (group != 32 && group != 64 && group != 128) || K % group) return (int)hipErrorInvalidValue;
  const long long tiles = (N + L4_TILE - 1) / L4_TILE, blocks = (K + L4_K - 1) / L4_K, groups = K / group;
  const int in_block = L4_K / group;
  const long long total = tiles * blocks * 256, per = tiles * blocks * in_block * 16;
  if ((total + 255) / 256 > 1LL << 30) return (int)hipErrorInvalidValue;
  hipLaunchKernelGGL(shuffle4_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st, (const unsigned char*)codes, (unsigned*)dst, N, K,
                     (int)blocks, total);
  hipLaunchKernelGGL((shuffle4_groups_kernel<bf16_t, true>), dim3((unsigned)((per + 255) / 256)), dim3(256), 0, st, (const bf16_t*)scales,
                     (bf16_t*)dst_scales, N, (int)groups, in_block, (int)blocks, per);
  if (zeros)
    hipLaunchKernelGGL((shuffle4_groups_kernel<unsigned char, false>), dim3((unsigned)((per + 255) / 256)), dim3(256), 0, st,
                       (const unsigned char*)zeros, (unsigned char*)dst_zeros, N, (int)groups, in_block, (int)blocks, per);
  return (int)hipGetLastError();
}

struct Linear4Args {
  const bf16_t* x;
  long long ldx;
  const l4_u4* w;
  const bf16_t* scales;
  const unsigned char* zeros;
  const bf16_t* bias;
  bf16_t* y;
  long long ldy;
  int M, N, K, parts;
  float* ws;
  int* tickets;
};

// MT: tiles of 16 rows of x; FT: tiles of features of a wave, which share its x; GS: MFMAs (of 32 columns) a group.
template <int FT, int GS> struct L4Block {
  static constexpr int NG = 4 / GS;
  l4_u4 c[FT];
  unsigned s[FT][2 * NG], z[FT];
};

// a wave-uniform address and a lane's offset, as the loads take them (64-bit sums a lane were a tenth of the loop)
template <typename T> __device__ __forceinline__ T l4_at(const void* base, unsigned off) {
  return *reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + off);
}

// Asks for block kb of tiles tile0 ..; blocks and tiles behind the last one read the last.
template <int FT, int GS, bool Z>
__device__ __forceinline__ void l4_load(L4Block<FT, GS>& b, const Linear4Args& A, int tile0, int tiles, int blocks, int kb, int lane) {
  constexpr int NG = 4 / GS;
  const int li = lane & 15, fq = lane >> 4;
  kb = min(kb, blocks - 1);
#pragma unroll
  for (int f = 0; f < FT; ++f) {
    const size_t at = (size_t)min(tile0 + f, tiles - 1) * blocks + kb;
    b.c[f] = l4_at<l4_u4>(A.w + at * 64, lane * 16);
    if constexpr (NG == 1) {
      const uint2 v = l4_at<uint2>(A.scales + at * 16, fq * 8);
      b.s[f][0] = v.x; b.s[f][1] = v.y;
    } else {
#pragma unroll
      for (int g = 0; g < NG; g += 2) {
        const uint4 v = l4_at<uint4>(A.scales + at * (16 * NG), fq * (8 * NG) + g * 8);
        b.s[f][2 * g] = v.x; b.s[f][2 * g + 1] = v.y; b.s[f][2 * g + 2] = v.z; b.s[f][2 * g + 3] = v.w;
      }
    }
    if constexpr (Z && NG == 1) b.z[f] = l4_at<unsigned char>(A.zeros + at * 16, li);
    if constexpr (Z && NG == 2) b.z[f] = l4_at<unsigned short>(A.zeros + at * 32, li * 2);
    if constexpr (Z && NG == 4) b.z[f] = l4_at<unsigned>(A.zeros + at * 64, li * 4);
  }
}

// acc += the block's products with x(t, s), columns 32 s .. of its tile t of rows. Behind K, in whole groups of scale zero, x(t, s) is
// any of the rows' own columns. AHEAD: a step's x is asked for before the products of the step before.
template <int MT, int FT, int GS, bool Z, bool AHEAD, typename X>
__device__ __forceinline__ void l4_work(float4v (&acc)[FT][MT], const L4Block<FT, GS>& b, unsigned magic, X&& x) {
  constexpr bool SHARE = !Z && MT <= 2;            // one MFMA of -136 for all features (nothing with four tiles of rows)
  constexpr unsigned M136 = 0xc308c308u;          // -136
  const float4v zero = {0.f, 0.f, 0.f, 0.f};
  float4v part[FT][MT], less[MT];
  bf16x8 ahead[MT];
  if constexpr (AHEAD) {
#pragma unroll
    for (int t = 0; t < MT; ++t) ahead[t] = x(t, 0);
  }
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int g = s / GS;
    bf16x8 xs[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xs[t] = AHEAD ? ahead[t] : x(t, s);
    if constexpr (AHEAD) {
      if (s < 3) {
#pragma unroll
        for (int t = 0; t < MT; ++t) ahead[t] = x(t, s + 1);
      }
    }
    __builtin_amdgcn_sched_barrier(0);            // steps one after the other: mixed, they hold more registers and wait for more at once
    if constexpr (SHARE) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
        less[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, l4_u4{M136, M136, M136, M136}), xs[t], s % GS == 0 ? zero : less[t],
                                                          0, 0, 0);
    }
#pragma unroll
    for (int f = 0; f < FT; ++f) {
      l4_u4 w, minus = {M136, M136, M136, M136};
      if constexpr (Z) {
        const unsigned z = (b.z[f] >> (8 * g)) & 255u, m = z | z << 16 | 0xc300c300u;
        minus = l4_u4{m, m, m, m};
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) w[p] = ((b.c[f][s] >> (4 * p)) & 0x000f000fu) | magic;
      if constexpr (!SHARE) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
          part[f][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, minus), xs[t], s % GS == 0 ? zero : part[f][t], 0, 0, 0);
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
        part[f][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), xs[t], SHARE && s % GS == 0 ? zero : part[f][t], 0, 0, 0);
      if (s % GS == GS - 1) {
        const unsigned s0 = b.s[f][2 * g], s1 = b.s[f][2 * g + 1];
        const float4v scale = {__uint_as_float(s0 << 16), __uint_as_float(s0 & 0xffff0000u), __uint_as_float(s1 << 16), __uint_as_float(s1 & 0xffff0000u)};
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[f][t][j] = fmaf(scale[j], SHARE ? part[f][t][j] + less[t][0] : part[f][t][j], acc[f][t][j]);   // less: all rows alike
      }
    }
  }
}

__device__ __forceinline__ unsigned l4_magic() {   // in a vector register: an AND-OR takes one constant from elsewhere
  unsigned magic = 0x43004300u;
  asm volatile("" : "+v"(magic));
  return magic;
}

// four features n .. of a row of y
__device__ __forceinline__ void l4_put(const Linear4Args& A, int row, int n, float4v o) {
  if (row >= A.M) return;
  bf16_t* y = A.y + (size_t)row * A.ldy + n;
  if (n + 4 <= A.N && (((size_t)A.y | (size_t)A.ldy * 2) & 7) == 0) {
    if (A.bias) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += bf2f(A.bias[n + j]);
    }
    *reinterpret_cast<uint2*>(y) = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
  } else {
    for (int j = 0; j < 4; ++j)
      if (n + j < A.N) y[j] = f2bf(o[j] + (A.bias ? bf2f(A.bias[n + j]) : 0.f));
  }
}

// Few rows: the waves of a workgroup share its features and divide K; they meet in LDS. A block's codes, scales, zeros and x
// are asked for while the block before is worked on.
template <int MT, int FT, int GS, bool Z, int NW>
__global__ __launch_bounds__(NW * 64) void linear4_kernel(Linear4Args A) {
  struct Block : L4Block<FT, GS> { bf16x8 x[MT][4]; };
  __shared__ float4v sums[NW][FT][MT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, fq = lane >> 4;
  const int tiles = (A.N + L4_TILE - 1) / L4_TILE, tile0 = blockIdx.x * FT;
  const int blocks = (A.K + L4_K - 1) / L4_K;
  const bf16_t* xp[MT];                           // rows behind the last one read the last
#pragma unroll
  for (int t = 0; t < MT; ++t) xp[t] = A.x + (size_t)min(16 * t + li, A.M - 1) * A.ldx + 8 * fq;
  const unsigned magic = l4_magic();
  const float4v zero = {0.f, 0.f, 0.f, 0.f};
  float4v acc[FT][MT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[f][t] = zero;
  auto load = [&](Block& b, int kb) __attribute__((always_inline)) {
    l4_load<FT, GS, Z>(b, A, tile0, tiles, blocks, kb, lane);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int s = 0; s < 4; ++s) b.x[t][s] = *reinterpret_cast<const bf16x8*>(xp[t] + min(min(kb, blocks - 1) * L4_K + 32 * s, A.K - 32));
  };
  auto work = [&](const Block& b) __attribute__((always_inline)) {
    l4_work<MT, FT, GS, Z, false>(acc, b, magic, [&](int t, int s) __attribute__((always_inline)) { return b.x[t][s]; });
  };
  if (wave < blocks) {
    Block a, b;
    load(a, wave);
    for (int kb = wave; kb < blocks; kb += 2 * NW) {
      load(b, kb + NW);
      work(a);
      if (kb + NW >= blocks) break;
      load(a, kb + 2 * NW);
      work(b);
    }
  }
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) sums[wave][f][t][lane] = acc[f][t];
  __syncthreads();
  for (int id = tid; id < FT * MT * 64; id += NW * 64) {
    const int f = id / (MT * 64), t = (id >> 6) % MT, l = id & 63;
    float4v o = zero;
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const float4v a = sums[v][f][t][l];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += a[j];
    }
    l4_put(A, 16 * t + (l & 15), (tile0 + f) * L4_TILE + 4 * (l >> 4), o);
  }
}

// Loads that go to LDS, a lane's bytes at dst + 16 lane (4 lane); the s_nops are the distances that m0 and a scalar register written
// by a vector instruction need.
__device__ __forceinline__ void l4_lds16(const void* base, unsigned off, unsigned dst) {   // base wave-uniform
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void l4_lds16(const void* at, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(at) : "memory", "m0");
}
__device__ __forceinline__ void l4_lds4(const void* at, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(dst), "v"(at) : "memory", "m0");
}

// More rows, 16 MT of them a workgroup: its four waves have FT tiles of features each and share the rows' x. All goes to LDS
// without registers, in a ring of R blocks (of x, a chunk of 8 columns lies at its number XOR the row's, so that the 16 rows of a
// fragment are in different banks). K is divided among `parts` workgroups; the last of them to arrive adds up what all have
// left, in order.
// Bound by its waves' issue, a SIMD's MFMAs (two for each step where zeros differ), and what each block waits for the one barrier: 64 rows
// x 28672 x 4096 37 us where the bytes take 13, 32 rows 25, 64 x 4096 x 4096 10.1, 32 x 4096 x 14336 14. (Each wave reading x from L2
// itself, K divided within a workgroup: 46, 30, 17.7, 31; x staged through registers, a block ahead: 39, 26, 13, 19; a ring of four
// blocks leaves room for fewer workgroups: 42 for the first.)
template <int MT, int FT, int GS, bool Z> struct L4Rows {
  static constexpr int R = MT == 2 ? 3 : 2;      // blocks of the ring
  static constexpr int NG = 4 / GS, X = MT * 4096, S = FT * 1024, ZS = S + FT * 32 * NG, MINE = ZS + (Z ? FT * 16 * NG : 0), STAGE = X + 4 * MINE;
  static constexpr int LOADS = MT + FT + 1 + Z;   // of a wave, a block
  static_assert(FT * 8 * NG <= 64 && MINE % 16 == 0, "one load for the scales, aligned reads");
};

template <int MT, int FT, int GS, bool Z>
__global__ __launch_bounds__(256, 2) void linear4_rows_kernel(Linear4Args A) {
  using L = L4Rows<MT, FT, GS, Z>;
  constexpr int NG = L::NG, R = L::R;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[R * L::STAGE];
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, fq = lane >> 4;
  const int tiles = (A.N + L4_TILE - 1) / L4_TILE, tile0 = (blockIdx.x * 4 + wave) * FT, m0 = blockIdx.y * (16 * MT);
  const int blocks = (A.K + L4_K - 1) / L4_K, share = (blocks + A.parts - 1) / A.parts, kb0 = blockIdx.z * share, kb1 = min(kb0 + share, blocks);
  const unsigned base = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char*)lds;
  // rows, tiles and blocks behind the last one read the last
  const int row = tid >> 4, col = ((tid & 15) ^ row) * 8;
  const bf16_t* xp[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xp[t] = A.x + (size_t)min(m0 + 16 * t + row, A.M - 1) * A.ldx;
  const l4_u4* wp[FT];
#pragma unroll
  for (int f = 0; f < FT; ++f) wp[f] = A.w + (size_t)min(tile0 + f, tiles - 1) * blocks * 64;
  const char* sp = (const char*)A.scales + (size_t)min(tile0 + lane / (8 * NG), tiles - 1) * blocks * (32 * NG) + lane % (8 * NG) * 4;
  const char* zp = (const char*)A.zeros + (size_t)min(tile0 + lane / (4 * NG), tiles - 1) * blocks * (16 * NG) + lane % (4 * NG) * 4;
  auto ask = [&](int kb, int stage) __attribute__((always_inline)) {
    kb = min(kb, blocks - 1);
    const unsigned at = base + stage * L::STAGE, mine = at + L::X + wave * L::MINE;
    const int c = min(kb * L4_K + col, A.K - 8);
#pragma unroll
    for (int t = 0; t < MT; ++t) l4_lds16(xp[t] + c, at + t * 4096 + wave * 1024);
#pragma unroll
    for (int f = 0; f < FT; ++f) l4_lds16(wp[f] + (size_t)kb * 64, lane * 16, mine + f * 1024);
    if (lane < FT * 8 * NG) l4_lds4(sp + (size_t)kb * (32 * NG), mine + L::S);
    if constexpr (Z) {
      if (lane < FT * 4 * NG) l4_lds4(zp + (size_t)kb * (16 * NG), mine + L::ZS);
    }
  };
  const unsigned magic = l4_magic();
  const float4v zero = {0.f, 0.f, 0.f, 0.f};
  float4v acc[FT][MT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[f][t] = zero;
#pragma unroll
  for (int i = 0; i < R - 1; ++i) ask(kb0 + i, i);
  int stage = 0;
  for (int kb = kb0; kb < kb1; ++kb) {
    // this wave's loads of the block have arrived, then the others', and all have read the block before, whose place is free
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((R - 2) * L::LOADS) : "memory");
    __syncthreads();
    ask(kb + R - 1, stage == 0 ? R - 1 : stage - 1);
    const unsigned char *at = lds + stage * L::STAGE, *mine = at + L::X + wave * L::MINE;
    L4Block<FT, GS> b;
#pragma unroll
    for (int f = 0; f < FT; ++f) {
      b.c[f] = *reinterpret_cast<const l4_u4*>(mine + f * 1024 + lane * 16);
      const unsigned* s = reinterpret_cast<const unsigned*>(mine + L::S + f * (32 * NG) + fq * (8 * NG));
#pragma unroll
      for (int g = 0; g < 2 * NG; ++g) b.s[f][g] = s[g];
      const unsigned char* z = mine + L::ZS + f * (16 * NG) + li * NG;
      if constexpr (Z && NG == 1) b.z[f] = *z;
      if constexpr (Z && NG == 2) b.z[f] = *reinterpret_cast<const unsigned short*>(z);
      if constexpr (Z && NG == 4) b.z[f] = *reinterpret_cast<const unsigned*>(z);
    }
    l4_work<MT, FT, GS, Z, true>(acc, b, magic, [&](int t, int s) __attribute__((always_inline)) {
      return *reinterpret_cast<const bf16x8*>(at + (t * 16 + li) * 256 + ((4 * s + fq) ^ li) * 16);
    });
    stage = stage == R - 1 ? 0 : stage + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no load is under way to LDS that has another owner
  if (A.parts > 1) {
    constexpr int PER = 4 * FT * MT * 1024;       // bytes of a part: a lane's sums as it has them
    const size_t unit = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(A.ws + unit * A.parts * (PER / 4), 0, A.parts * PER, 0x00020000);
    const int at = (wave * FT * MT * 64 + lane) * 16;
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int t = 0; t < MT; ++t)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(l4_u4, acc[f][t]), rs, blockIdx.z * PER + at + (f * MT + t) * 1024, 0, 16);
    // this wave's stores have arrived, then the others'
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0) {
      const int n = __hip_atomic_fetch_add(A.tickets + unit * TICKET, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (n == A.parts - 1) __hip_atomic_store(A.tickets + unit * TICKET, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = n == A.parts - 1;
    }
    __syncthreads();
    if (!last) return;
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[f][t] = zero;
    constexpr int OB = 16 / (FT * MT);            // parts asked for together
    for (int p0 = 0; p0 < A.parts; p0 += OB) {
      float4v v[OB][FT][MT];
#pragma unroll
      for (int i = 0; i < OB; ++i)
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
          for (int t = 0; t < MT; ++t)            // behind the last part: the buffer's end, zeros
            v[i][f][t] = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(rs, (p0 + i) * PER + at + (f * MT + t) * 1024, 0, 16));
#pragma unroll
      for (int i = 0; i < OB; ++i)
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[f][t][j] += v[i][f][t][j];
    }
  }
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) l4_put(A, m0 + 16 * t + li, (tile0 + f) * L4_TILE + 4 * fq, acc[f][t]);
}

template <int MT, int FT, int GS, int NW> static void l4_go(const Linear4Args& a, hipStream_t st) {
  const dim3 grid(((a.N + L4_TILE - 1) / L4_TILE + FT - 1) / FT);
  if (a.zeros) hipLaunchKernelGGL((linear4_kernel<MT, FT, GS, true, NW>), grid, dim3(NW * 64), 0, st, a);
  else hipLaunchKernelGGL((linear4_kernel<MT, FT, GS, false, NW>), grid, dim3(NW * 64), 0, st, a);
}

template <int MT, int FT, int GS> static void l4_rows(const Linear4Args& a, hipStream_t st) {
  const dim3 grid(((a.N + L4_TILE - 1) / L4_TILE + 4 * FT - 1) / (4 * FT), (a.M + 16 * MT - 1) / (16 * MT), a.parts);
  if (a.zeros) hipLaunchKernelGGL((linear4_rows_kernel<MT, FT, GS, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((linear4_rows_kernel<MT, FT, GS, false>), grid, dim3(256), 0, st, a);
}

// Features of a wave and waves of a workgroup. A wave of four tiles reads its x a quarter as often and has four kilobytes under
// way; of one, there are four times as many workgroups. us by (tiles a wave, waves), cold weights, launches in a replayed graph:
// 1 row x 28672 x 4096 (groups of 128) 20.8 (1, 8), 17.1 (2, 8), 16.6 (4, 8), 15.0 (4, 4); 8 rows (64, zeros) 28.2, 20.8, 19.9, 17.0;
// 4 x 12288 x 4096 11.6, 10.8, 9.8, 9.5; 4 x 8192 x 4096 7.7, 6.3, 8.4, 9.0; 1 x 4096 x 4096 4.4, 5.3, 7.4, 7.7. Two tiles of rows come
// with few features: 32 x 4096 x 4096 11.9, 12.3, 13.9, 12.8.
template <int GS> static void l4_features(const Linear4Args& a, hipStream_t st) {
  const int tiles = (a.N + L4_TILE - 1) / L4_TILE;
  if (a.M > 16) return l4_go<2, 1, GS, 8>(a, st);
  if (tiles >= 640) return l4_go<1, 4, GS, 4>(a, st);
  if (tiles >= 384) return l4_go<1, 2, GS, 8>(a, st);
  l4_go<1, 1, GS, 8>(a, st);
}

template <int GS> static void l4_group(const Linear4Args& a, int features, hipStream_t st) {
  if (features == 0) return l4_features<GS>(a, st);
  if (a.M <= 32) features == 1 ? l4_rows<2, 1, GS>(a, st) : l4_rows<2, 2, GS>(a, st);
  else features == 1 ? l4_rows<4, 1, GS>(a, st) : l4_rows<4, 2, GS>(a, st);
}

// `features`: tiles of features a wave of the kernel for more rows, in `parts` of K; 0: the kernel for few rows (up to 32).
extern "C" int loqa_linear4(const void* x, long ldx, const void* w, const void* scales, const void* zeros, const void* bias, void* y, long ldy, int M,
                            int N, int K, int group, int features, int parts, void* ws, long ws_floats, void* tickets, long n_tickets, hipStream_t st) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || (group != 32 && group != 64 && group != 128) || K % group || ldx < 0 || ldx % 8 || ((size_t)x & 15)) return (int)hipErrorInvalidValue;
  if (features < 0 || features > 2) return (int)hipErrorInvalidValue;
  if (parts < 1 || (features == 0 && (M > 32 || parts > 1))) return (int)hipErrorInvalidValue;
  const long tiles = (N + (long)L4_TILE - 1) / L4_TILE, blocks = (K + (long)L4_K - 1) / L4_K;
  if (features) {
    const int mt = M <= 32 ? 2 : 4;
    const long across = (tiles + 4 * features - 1) / (4 * features), rows = (M + 16L * mt - 1) / (16 * mt);
    if (rows > 65535 || parts > 64 || (blocks + parts - 1) / parts * (parts - 1) >= blocks) return (int)hipErrorInvalidValue;   // an empty part
    if (parts > 1 && (!ws || !tickets || across * rows > n_tickets || across * rows * parts > ws_floats / (1024L * features * mt)))
      return (int)hipErrorInvalidValue;
  }
  const Linear4Args a{(const bf16_t*)x, ldx, (const l4_u4*)w, (const bf16_t*)scales, (const unsigned char*)zeros, (const bf16_t*)bias, (bf16_t*)y, ldy,
                      M, N, K, parts, (float*)ws, (int*)tickets};
  if (group == 32) l4_group<1>(a, features, st);
  else if (group == 64) l4_group<2>(a, features, st);
  else l4_group<4>(a, features, st);
  return (int)hipGetLastError();
}
