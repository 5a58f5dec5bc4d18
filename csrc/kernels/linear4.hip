// y = x W^T + bias for a few rows of x, W [N, K] in 4 bits: W[n, k] = (c[n, k] - z[n, k / g]) s[n, k / g], codes c and
// zeros z in 0 .. 15 (z = 8 where there are none), s in bf16, groups of g = 32, 64 or 128 columns.
//
// Bound by the bytes of the codes, which each wave streams as whole kilobytes: 16 features by 128 columns, laid out
// once as the MFMA wants them (shuffle4 below), a lane's 16 bytes the codes of its feature for four MFMAs. Codes become
// bf16 without arithmetic: 0x4300 | c is 128 + c exactly, so a pair of them costs an AND-OR and a shift. The group's
// sum then is
//
//   sum_k (128 + c) x  =  sum_k (c - z) x  +  (128 + z) sum_k x,
//
// of which the second part is taken off in f32, with sum_k x from one more MFMA of ones (shared by a wave's
// features), before the scale; products of whole numbers up to 143 with bf16 are exact, and what f32 sums lose, 2^-24
// of terms up to 143 |x| where the result's own are up to 15 |x|, is far below the result's rounding to bf16.
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

// [N, groups] -> [tile][group][16], zeros past N
template <typename T> __global__ __launch_bounds__(256) void shuffle4_groups_kernel(const T* src, T* dst, int N, int groups, long long total) {
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const long long tg = id >> 4;
  const int n = (int)(tg / groups) * L4_TILE + (int)(id & 15), g = (int)(tg % groups);
  dst[id] = n < N ? src[(size_t)n * groups + g] : (T)0;
}

extern "C" int loqa_shuffle4(const void* codes, const void* scales, const void* zeros, void* dst, void* dst_scales, void* dst_zeros, int N, int K,
                             int group, hipStream_t st) {
  if (N <= 0 || K <= 0 || K % 32 || (group != 32 && group != 64 && group != 128) || K % group) return (int)hipErrorInvalidValue;
  const long long tiles = (N + L4_TILE - 1) / L4_TILE, blocks = (K + L4_K - 1) / L4_K, groups = K / group;
  const long long total = tiles * blocks * 256, per = tiles * groups * 16;
  if ((total + 255) / 256 > 1LL << 30) return (int)hipErrorInvalidValue;
  hipLaunchKernelGGL(shuffle4_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st, (const unsigned char*)codes, (unsigned*)dst, N, K,
                     (int)blocks, total);
  hipLaunchKernelGGL((shuffle4_groups_kernel<bf16_t>), dim3((unsigned)((per + 255) / 256)), dim3(256), 0, st, (const bf16_t*)scales,
                     (bf16_t*)dst_scales, N, (int)groups, per);
  if (zeros)
    hipLaunchKernelGGL((shuffle4_groups_kernel<unsigned char>), dim3((unsigned)((per + 255) / 256)), dim3(256), 0, st, (const unsigned char*)zeros,
                       (unsigned char*)dst_zeros, N, (int)groups, per);
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

// MT: tiles of 16 rows of x; GS: MFMAs (of 32 columns) a group
template <int MT, int GS, bool Z, int NW>
__global__ __launch_bounds__(NW * 64) void linear4_kernel(Linear4Args A) {
  __shared__ float4v sums[NW][MT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, li = lane & 15, fq = lane >> 4;
  const int tile = blockIdx.x, m0 = blockIdx.y * (16 * MT), blocks = (A.K + L4_K - 1) / L4_K, groups = A.K / (32 * GS);
  const l4_u4* w = A.w + ((size_t)tile * blocks) * 64 + lane;
  const bf16_t* sp = A.scales + (size_t)tile * groups * 16 + 4 * fq;
  const unsigned char* zp = A.zeros + (size_t)tile * groups * 16 + 4 * fq;
  const bf16_t* xp[MT];                           // rows behind the last one read the last
#pragma unroll
  for (int t = 0; t < MT; ++t) xp[t] = A.x + (size_t)min(m0 + 16 * t + li, A.M - 1) * A.ldx + 8 * fq;
  bf16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (__bf16)1.0f;
  const float4v zero = {0.f, 0.f, 0.f, 0.f};
  float4v acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = zero;
  for (int kb = wave; kb < blocks; kb += NW) {
    const l4_u4 c = w[(size_t)kb * 64];
    float4v part[MT], xs[MT];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int k = kb * L4_K + 32 * s;
      if (k >= A.K) break;                        // uniform
      if (s % GS == 0) {
#pragma unroll
        for (int t = 0; t < MT; ++t) part[t] = xs[t] = zero;
      }
      l4_u4 b;
#pragma unroll
      for (int p = 0; p < 4; ++p) b[p] = ((c[s] >> (4 * p)) & 0x000f000fu) | 0x43004300u;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const bf16x8 xf = *reinterpret_cast<const bf16x8*>(xp[t] + k);
        part[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), xf, part[t], 0, 0, 0);
        xs[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, xf, xs[t], 0, 0, 0);
      }
      if (s % GS == GS - 1) {
        const int g = k / (32 * GS);
        const uint2 sc = *reinterpret_cast<const uint2*>(sp + (size_t)g * 16);
        const float4v scale = {__uint_as_float(sc.x << 16), __uint_as_float(sc.x & 0xffff0000u), __uint_as_float(sc.y << 16), __uint_as_float(sc.y & 0xffff0000u)};
        float4v off = {136.f, 136.f, 136.f, 136.f};
        if constexpr (Z) {
          const unsigned z = *reinterpret_cast<const unsigned*>(zp + (size_t)g * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) off[j] = 128.f + (float)((z >> (8 * j)) & 255u);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[t][j] = fmaf(scale[j], fmaf(-off[j], xs[t][j], part[t][j]), acc[t][j]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) sums[wave][t][lane] = acc[t];
  __syncthreads();
  for (int id = tid; id < MT * 64; id += NW * 64) {
    const int t = id >> 6, l = id & 63, row = m0 + 16 * t + (l & 15), n = tile * L4_TILE + 4 * (l >> 4);
    float4v o = zero;
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const float4v a = sums[v][t][l];
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

template <int MT, int GS> static void l4_go(const Linear4Args& a, hipStream_t st) {
  constexpr int NW = 8;
  const dim3 grid((a.N + L4_TILE - 1) / L4_TILE, (a.M + 16 * MT - 1) / (16 * MT));
  if (a.zeros) hipLaunchKernelGGL((linear4_kernel<MT, GS, true, NW>), grid, dim3(NW * 64), 0, st, a);
  else hipLaunchKernelGGL((linear4_kernel<MT, GS, false, NW>), grid, dim3(NW * 64), 0, st, a);
}

template <int MT> static void l4_group(const Linear4Args& a, int group, hipStream_t st) {
  if (group == 32) l4_go<MT, 1>(a, st);
  else if (group == 64) l4_go<MT, 2>(a, st);
  else l4_go<MT, 4>(a, st);
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
