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
// eight rows in groups of 64 with zeros 20 us, 17 now.)
// The waves of a workgroup share its features and divide K; they meet in LDS.
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
  int M, N, K;
};

// MT: tiles of 16 rows of x; FT: tiles of features of a wave, which share its x; GS: MFMAs (of 32 columns) a group. A block's
// codes, scales and zeros are asked for while the block before is worked on, and the x of up to two tiles of rows.
template <int MT, int FT, int GS, bool Z> struct L4Block {
  static constexpr int NG = 4 / GS;
  static constexpr bool SHARE = !Z && MT <= 2;     // one MFMA of -136 for all features (with four tiles of rows its registers cost more)
  l4_u4 c[FT];
  unsigned s[FT][2 * NG], z[FT];
  bf16x8 x[MT <= 2 ? MT : 1][4];
};

// a wave-uniform address and a lane's offset, as the loads take them (64-bit sums a lane were a tenth of the loop)
template <typename T> __device__ __forceinline__ T l4_at(const void* base, unsigned off) {
  return *reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + off);
}

template <int MT, int FT, int GS, bool Z, int NW>
__global__ __launch_bounds__(NW * 64) void linear4_kernel(Linear4Args A) {
  using Block = L4Block<MT, FT, GS, Z>;
  constexpr int NG = Block::NG;
  constexpr bool SHARE = Block::SHARE;
  __shared__ float4v sums[NW][FT][MT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, fq = lane >> 4;
  const int tiles = (A.N + L4_TILE - 1) / L4_TILE, tile0 = blockIdx.x * FT, m0 = blockIdx.y * (16 * MT);
  const int blocks = (A.K + L4_K - 1) / L4_K;
  const bf16_t* xp[MT];                           // rows behind the last one read the last
#pragma unroll
  for (int t = 0; t < MT; ++t) xp[t] = A.x + (size_t)min(m0 + 16 * t + li, A.M - 1) * A.ldx + 8 * fq;
  unsigned magic = 0x43004300u;                   // in a vector register: an AND-OR takes one constant from elsewhere
  asm volatile("" : "+v"(magic));
  const float4v zero = {0.f, 0.f, 0.f, 0.f};
  float4v acc[FT][MT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[f][t] = zero;
  auto xread = [&](int t, int kb, int s) __attribute__((always_inline)) { return *reinterpret_cast<const bf16x8*>(xp[t] + min(kb * L4_K + 32 * s, A.K - 32)); };
  auto load = [&](Block& b, int kb) __attribute__((always_inline)) {
    kb = min(kb, blocks - 1);
#pragma unroll
    for (int f = 0; f < FT; ++f) {                // tiles behind the last one read the last
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
    if constexpr (MT <= 2) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int s = 0; s < 4; ++s) b.x[t][s] = xread(t, kb, s);
    }
  };
  auto work = [&](const Block& b, int kb) __attribute__((always_inline)) {
    bf16x8 x[MT][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if constexpr (MT <= 2) x[t][s] = b.x[t][s];
        else x[t][s] = xread(t, kb, s);
      }
    float4v part[FT][MT], less[MT];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (kb * L4_K + 32 * s >= A.K) break;       // uniform
      const int g = s / GS;
      constexpr unsigned M136 = 0xc308c308u;      // -136
      if constexpr (SHARE) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
          less[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, l4_u4{M136, M136, M136, M136}), x[t][s],
                                                            s % GS == 0 ? zero : less[t], 0, 0, 0);
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
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if constexpr (!SHARE)
            part[f][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, minus), x[t][s], s % GS == 0 ? zero : part[f][t], 0, 0, 0);
          part[f][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), x[t][s], SHARE && s % GS == 0 ? zero : part[f][t], 0, 0, 0);
        }
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
  };
  if (wave < blocks) {
    Block a, b;
    load(a, wave);
    for (int kb = wave; kb < blocks; kb += 2 * NW) {
      load(b, kb + NW);
      work(a, kb);
      if (kb + NW >= blocks) break;
      load(a, kb + 2 * NW);
      work(b, kb + NW);
    }
  }
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < MT; ++t) sums[wave][f][t][lane] = acc[f][t];
  __syncthreads();
  for (int id = tid; id < FT * MT * 64; id += NW * 64) {
    const int f = id / (MT * 64), t = (id >> 6) % MT, l = id & 63, row = m0 + 16 * t + (l & 15), n = (tile0 + f) * L4_TILE + 4 * (l >> 4);
    float4v o = zero;
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const float4v a = sums[v][f][t][l];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += a[j];
    }
    if (row >= A.M) continue;
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
}

template <int MT, int FT, int GS, int NW> static void l4_go(const Linear4Args& a, hipStream_t st) {
  const int tiles = (a.N + L4_TILE - 1) / L4_TILE;
  const dim3 grid((tiles + FT - 1) / FT, (a.M + 16 * MT - 1) / (16 * MT));
  if (a.zeros) hipLaunchKernelGGL((linear4_kernel<MT, FT, GS, true, NW>), grid, dim3(NW * 64), 0, st, a);
  else hipLaunchKernelGGL((linear4_kernel<MT, FT, GS, false, NW>), grid, dim3(NW * 64), 0, st, a);
}

// Features of a wave and waves of a workgroup. A wave of four tiles reads its x a quarter as often and has four kilobytes under
// way; of one, there are four times as many workgroups. us by (tiles a wave, waves), cold weights, launches in a replayed graph:
// 1 row x 28672 x 4096 (groups of 128) 20.8 (1, 8), 17.1 (2, 8), 16.6 (4, 8), 15.0 (4, 4); 8 rows (64, zeros) 28.2, 20.8, 19.9, 17.0;
// 4 x 12288 x 4096 11.6, 10.8, 9.8, 9.5; 4 x 8192 x 4096 7.7, 6.3, 8.4, 9.0; 1 x 4096 x 4096 4.4, 5.3, 7.4, 7.7; 32 rows x 14336 x
// 4096 39.8, 23.4, 15.5, 14.0; 64 rows 64.2, 37.3, 23.4, 27.6, x 4096 x 4096 17.7, 18.5, 20.8, 25.8; 18 rows x 8656 x
// 8448 38.2, 29.9, 21.2, 19.8, 32 x 4096 x 4096 11.9, 12.3, 13.9, 12.8.
template <int MT, int GS> static void l4_features(const Linear4Args& a, hipStream_t st) {
  const int tiles = (a.N + L4_TILE - 1) / L4_TILE;
  if (tiles >= (MT == 2 ? 384 : 640)) return l4_go<MT, 4, GS, MT <= 2 ? 4 : 8>(a, st);
  if (tiles >= 384) return l4_go<MT, 2, GS, 8>(a, st);
  l4_go<MT, 1, GS, 8>(a, st);
}

template <int MT> static void l4_group(const Linear4Args& a, int group, hipStream_t st) {
  if (group == 32) l4_features<MT, 1>(a, st);
  else if (group == 64) l4_features<MT, 2>(a, st);
  else l4_features<MT, 4>(a, st);
}

extern "C" int loqa_linear4(const void* x, long ldx, const void* w, const void* scales, const void* zeros, const void* bias, void* y, long ldy, int M,
                            int N, int K, int group, hipStream_t st) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || (group != 32 && group != 64 && group != 128) || K % group || ldx < 0 || ldx % 8 || ((size_t)x & 15) || (M + 63) / 64 > 65535)
    return (int)hipErrorInvalidValue;
  const Linear4Args a{(const bf16_t*)x, ldx, (const l4_u4*)w, (const bf16_t*)scales, (const unsigned char*)zeros, (const bf16_t*)bias, (bf16_t*)y, ldy,
                      M, N, K};
  if (M <= 16) l4_group<1>(a, group, st);
  else if (M <= 32) l4_group<2>(a, group, st);
  else l4_group<4>(a, group, st);
  return (int)hipGetLastError();
}
