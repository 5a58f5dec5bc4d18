// Attention off the paged cache in 8 bits (cache8.h). Rows r of a feed are its tokens times the G query heads of a kv
// head, token r / G and head r % G: every key and value is read, and widened to f16, once for all of them.
//
//   x_j = q . k_j (f16 MFMAs, f32 sums),  s_j = scale log2(e) ks x_j,  o = sum_j 2^(s_j) vs v_j / sum_j 2^(s_j)
//
// with ks, vs of a key's page. The values' scale goes into the exponent: t_j = s_j + log2(vs), weights w_j = 2^(t_j - m)
// are what the codes of v are summed up with, and the denominator is sum_j w_j / vs in f32. The reference m of a row starts 2^7 below its
// largest t_j and follows it within a factor of 2^8, so weights reach 2^15 and are f16 without a range of their own: 11 bits each, under
// 2^-14 an absolute 2^-25. The largest is 2^7 or more, so what becomes zero there is under 2^-32 of it, and n such keys, which the f32
// denominator still counts, lose 2^-32 n (with a reference at the largest, 2^-25 n: 3 % of a million). With a reference that never lags, some
// row of a wave has a new maximum in nearly every tile, and rescaling is a tenth of a tile's instructions. The denominator is
// summed up 2^7 smaller, for the room that scales of 2^-100 leave it. Queries enter as f16 times a power of two of
// the row that puts its largest entry in 2^14 .. 2^15: bf16's 8 bits are exact down to 2^-28 of it.
//
// Rows that see no key (a position before the first) give zeros; keys of pages that do not exist count as masked.
#include "cache8.h"
#include "flash_pipe.h"

#define A8_NONE -3.0e38f                           // a row's reference before its first key
#define A8_BELOW 7.f                               // of a largest score, the reference that it sets
#define A8_MOST 15.f                               // of a weight, as a power of two: then the reference moves
#define A8_DOWN 0.0078125f                         // 2^-7, of the denominator

struct Attn8Args {
  const bf16_t* q;
  long long ldq;
  const unsigned char *k, *v;
  const float *ks, *vs;
  const int *cu, *ctx, *bt;
  bf16_t* out;
  long long ldo;
  float* ws;                             // partials: [unit][part][rows][D + 2]
  int* tickets;
  int T, B, H, G, sh, n_blocks, max_blocks, max_q, parts, causal, row_blocks, each, fold;
  float scale_log2;
};

// a feed's metadata, whatever the numbers say: rows 0 .. T, keys that the table has
struct A8Feed { int q0, n, keys, past; };
__device__ __forceinline__ int a8_scalar(const int* p) { return *(const __attribute__((address_space(4))) int*)(size_t)p; }
__device__ __forceinline__ A8Feed a8_feed(const Attn8Args& A, int b) {
  A8Feed f;
  f.q0 = min(max(a8_scalar(A.cu + b), 0), A.T);
  const int n = min(max(a8_scalar(A.cu + b + 1), f.q0), A.T) - f.q0, L = a8_scalar(A.ctx + b);
  f.past = L - n;
  f.n = min(n, A.max_q);
  f.keys = (int)min((long long)max(L, 0), (long long)A.max_blocks << A.sh);
  return f;
}

// N pieces of eight entries of a query row, piece u at at(u), asked for together (rows at odd places entry by entry)
template <int N, typename At> __device__ __forceinline__ void a8_row(const Attn8Args& A, uint4 (&x)[N], At&& at) {
  if ((((size_t)A.q | (size_t)A.ldq * 2) & 15) == 0) {
#pragma unroll
    for (int u = 0; u < N; ++u) x[u] = *reinterpret_cast<const uint4*>(at(u));
  } else {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const bf16_t* p = at(u);
      unsigned w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = p[2 * i] | (unsigned)p[2 * i + 1] << 16;
      x[u] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// the f16 form of a row's pieces, times 2^e and its sign; top: the row's largest magnitude
template <int N> __device__ __forceinline__ float a8_top(const uint4 (&x)[N]) {
  float top = 0.f;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    float f[8];
    unpack8(x[u], f);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[i]));
  }
  return top;
}
template <int N> __device__ __forceinline__ void a8_queries(const uint4 (&x)[N], bool row, int e, bool minus, c8_h8 (&q)[N]) {
  const float by = !row ? 0.f : ldexpf(minus ? -1.f : 1.f, e);
#pragma unroll
  for (int u = 0; u < N; ++u) {
    float f[8];
    unpack8(x[u], f);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[u][i] = row ? (_Float16)(f[i] * by) : (_Float16)0.f;
  }
}

// the power of two that puts a largest magnitude into 2^14 .. 2^15, as an exponent (0 for a row of zeros)
__device__ __forceinline__ int a8_lift(float top) {
  return top > 0.f && top < INFINITY ? min(14 - (int)((__float_as_uint(top) >> 23) & 255) + 127, 126) : 0;
}

// ---- the partials of a unit's parts, joined by the last of them: [unit][part][R rows][D columns, then maximum and sum]. Written
// through and read past the caches: parts may run on different XCDs.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t a8_rsrc(const Attn8Args& A, size_t unit, int part, int rows, int D) {
  return __builtin_amdgcn_make_buffer_rsrc(A.ws + (unit * A.parts + part) * rows * (D + 2), 0, rows * (D + 2) * 4, 0x00020000);
}
typedef unsigned a8_u4 __attribute__((ext_vector_type(4)));
typedef unsigned a8_u2 __attribute__((ext_vector_type(2)));

// All of the workgroup's partials are on their way: whether it is the last of the n parts to arrive (then all of them are
// in memory). The wait is for this wave's stores, the barrier for the others'.
__device__ __forceinline__ bool a8_last(int* ticket, int n, int* flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const int t = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (t == n - 1) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = t == n - 1;
  }
  __syncthreads();
  return *flag != 0;
}

__device__ __forceinline__ void a8_put(bf16_t* at, const float4v& o, float l, bool whole) {
  const float inv = l == 0.f ? 0.f : 1.f / l;     // NaN stays
  const uint2 w = make_uint2(pack_bf16x2(o[0] * A8_DOWN * inv, o[1] * A8_DOWN * inv), pack_bf16x2(o[2] * A8_DOWN * inv, o[3] * A8_DOWN * inv));
  if (whole) {
    *reinterpret_cast<uint2*>(at) = w;
  } else {
    at[0] = (bf16_t)w.x; at[1] = (bf16_t)(w.x >> 16); at[2] = (bf16_t)w.y; at[3] = (bf16_t)(w.y >> 16);
  }
}

// Joins n parts of `rows` rows and writes them; NT threads, eight partials under way each. A thread has four columns of a row, and
// where there are threads left (few rows), as many of them share the parts as there are whole groups: they meet in LDS
// (at `room`, NT * 24 bytes), in order. (Two contexts of 27000 keys x 2 heads of 64 in 120 parts
// each 23.6 -> 15.4 us.)
template <int D, int R, int NT, typename Put>
__device__ __forceinline__ void a8_join(const Attn8Args& A, size_t unit, int n, int rows, float* room, Put&& put) {
  constexpr int OB = 8, PER = R * (D + 2) * 4;
  const auto rs = __builtin_amdgcn_make_buffer_rsrc(A.ws + unit * A.parts * R * (D + 2), 0, A.parts * PER, 0x00020000);
  auto sum = [&](int r, int c, int from, int to, float& ms, float& l, float4v& o) __attribute__((always_inline)) {
    ms = A8_NONE;
    l = 0.f;
    o = float4v{0.f, 0.f, 0.f, 0.f};
    for (int s0 = from; s0 < to; s0 += OB) {
      float4v v[OB];
      float2 ml[OB];
#pragma unroll
      for (int i = 0; i < OB; ++i) {
        const int at = min(s0 + i, to - 1) * PER;
        ml[i] = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(rs, at + (R * D + 2 * r) * 4, 0, 16));
        v[i] = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(rs, at + (r * D + c) * 4, 0, 16));
      }
      // all are asked for before the first is waited for
#pragma unroll
      for (int i = 0; i < OB; ++i) asm volatile("" : "+v"(ml[i].x), "+v"(ml[i].y), "+v"(v[i]));
      float mn = ms;
#pragma unroll
      for (int i = 0; i < OB; ++i) mn = fmaxf(mn, ml[i].x);
      const float a = exp2f(ms - mn);
      ms = mn;
      l *= a;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] *= a;
#pragma unroll
      for (int i = 0; i < OB; ++i) {
        if (s0 + i >= to) break;
        const float x = exp2f(ml[i].x - ms);
        l += x * ml[i].y;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += x * v[i][j];
      }
    }
  };
  const int items = rows * (D / 4), groups = n > OB ? max(1, min(NT / items, (n + OB - 1) / OB)) : 1;
  float ms, l;
  float4v o;
  if (groups == 1) {
    for (int id = threadIdx.x; id < items; id += NT) {
      sum(id / (D / 4), id % (D / 4) * 4, 0, n, ms, l, o);
      put(id / (D / 4), id % (D / 4) * 4, o, l);
    }
    return;
  }
  const int g = threadIdx.x / items, id = threadIdx.x - g * items, r = id / (D / 4), c = id % (D / 4) * 4;
  if (g < groups) {
    sum(r, c, n * g / groups, n * (g + 1) / groups, ms, l, o);
    float* at = room + threadIdx.x * 6;
    at[0] = ms; at[1] = l;
#pragma unroll
    for (int j = 0; j < 4; ++j) at[2 + j] = o[j];
  }
  __syncthreads();
  if (g > 0) return;
  for (int k = 1; k < groups; ++k) {
    const float* at = room + (k * items + id) * 6;
    const float mn = fmaxf(ms, at[0]), a = exp2f(ms - mn), x = exp2f(at[0] - mn);
    ms = mn;
    l = l * a + at[1] * x;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = o[j] * a + at[2 + j] * x;
  }
  put(r, c, o, l);
}

// ------------------------------------------------------------------ token steps
// RT tiles of 16 rows per kv head, one or two. A step reads every cached code once, so it is bound by the bytes a compute unit has
// under way: each wave streams tiles of 32 keys straight to its own ring of two in LDS, as the bf16 form does
// (attn_stream.hip), the scales of a tile's two pages with it. The waves of a workgroup take tiles in turn, the
// workgroups of a sequence parts of its keys. A tile is 8 KB to the bf16 form's 16 and as much work: page numbers are scalars
// that no wait precedes (kept in an array they went through LDS, and a tile waited for the next one's: 32 x 4000 keys x 8
// heads of 128 66 us), values are asked of LDS ahead of the exponentials. us, cold caches, pages of 16 (bf16 form): 32 x 4000 keys x 8
// heads of 128 50 (96), 5.0 TB/s; 1 x 100000 38, 5.4; 256 x 1000 92 (159); 8 x 600 10 (13); 1 x 600 6.8 (10.9); 64 x 300 13 (21); 8 x
// 1500 x 20 of 64 13 (19). Two tiles of rows share what is widened: 32 rows behind 1 x 30000 keys x 8 heads of 128 37 (the prompt form below
// 65), 16 x 4000 40 (56), 32 x 1000 20 (36). Four of them, with one workgroup a compute unit: 64 rows 62 (65), 76 (57), 33 (37); left out.
//
//   S^T = K Q^T   : 16 x 16 x 32 MFMAs; a lane reads 16 codes of a key at once, the K slots of two MFMAs
//   O^T += V^T P^T: eight keys of one column by a transposing read of bytes; P^T is the accumulator as it stands
#define A8_TILE 32
#define A8_WAVES 4
#define A8_LDS __attribute__((address_space(3)))
template <typename T> __device__ __forceinline__ A8_LDS T* a8_lds(unsigned at) { return (A8_LDS T*)(size_t)at; }
typedef int a8_v2i __attribute__((ext_vector_type(2)));

// 16 bytes a lane at rsrc + off to LDS at dst + 16 lane, zeros from out of range; the s_nop is the distance that a scalar
// register written by a vector instruction needs, and m0's
__device__ __forceinline__ void a8_load16(const a8_u4& rsrc, unsigned off, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(dst), "v"(off), "s"(rsrc) : "memory", "m0");
}
__device__ __forceinline__ void a8_load4(const float* at, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(dst), "v"(at) : "memory", "m0");
}
__device__ __forceinline__ a8_u4 a8_raw(const unsigned char* base, unsigned bytes) {
  const unsigned long long at = (unsigned long long)base;
  return a8_u4{(unsigned)__builtin_amdgcn_readfirstlane((int)at), (unsigned)__builtin_amdgcn_readfirstlane((int)(at >> 32)),
               (unsigned)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}
template <int N> __device__ __forceinline__ void a8_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// R: stages of a wave's ring; one where no wave has a second tile, so that twice as many workgroups fit a compute unit
template <int D, int R, int RT> struct A8Token {
  static constexpr int ROWS = 16 * RT;
  static constexpr int TB = A8_TILE * D, STAGE = 2 * TB + 256;         // K, V, a dword a lane of scales
  static constexpr int RING = R * STAGE;
  static constexpr int MERGE = A8_WAVES * ROWS * (D + 4 + 2) * 4 + 16;
  static constexpr int SMEM = A8_WAVES * RING > MERGE ? A8_WAVES * RING : MERGE;
  static constexpr int FIT = 163840 / SMEM < 4 ? 163840 / SMEM : 4;    // workgroups of a compute unit
};

__device__ __forceinline__ float a8_max16(float x) {    // over lane and lane ^ 16
  const a8_u2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float a8_sum16(float x) {
  const a8_u2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int D, int KIND, int R, int RT>
__global__ __launch_bounds__(A8_WAVES * 64, (A8Token<D, R, RT>::FIT)) void attn8_token_kernel(Attn8Args A) {
  using L = A8Token<D, R, RT>;
  constexpr int ROWS = L::ROWS;
  constexpr int LPR = D / 16, RPL = 64 / LPR, NL = A8_TILE / RPL;      // lanes a row, rows a load, loads of K (and of V)
  constexpr int NS = D / 64, ND = D / 16, LD = D + 4;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[L::SMEM];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, fq = lane >> 4;
  const int part = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, Gq = A.H / A.G;
  const A8Feed f = a8_feed(A, b);
  const int tiles = (f.keys + A8_TILE - 1) / A8_TILE, each = max((tiles + A.parts - 1) / A.parts, A8_WAVES);
  const int nparts = max((tiles + each - 1) / each, 1);
  if (f.n == 0 || part >= nparts) return;
  const int kend = min(f.keys, (part + 1) * each * A8_TILE), rows = f.n * Gq;
  const int kt0 = (part * each + wave) * A8_TILE;
  constexpr int STEP = A8_WAVES * A8_TILE;
  const int* bt = A.bt + (size_t)b * A.max_blocks;
  auto page_at = [&](int kt) { return a8_scalar(bt + min(kt >> A.sh, A.max_blocks - 1)); };
  // page numbers of the tile asked for next and of the one behind it
  int pa0 = page_at(kt0), pa1 = page_at(kt0 + 16), pb0 = R > 1 ? page_at(kt0 + STEP) : 0, pb1 = R > 1 ? page_at(kt0 + STEP + 16) : 0;

  // the queries of rows 16 r + li, asked for ahead of the first tile: K slots (fq, e) of MFMAs 2 s and 2 s + 1 are columns 64 s + 16 fq + e
  // and + 8 + e
  uint4 x[RT][2 * NS];
  int seen[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int at = 16 * r + li, tok = at / Gq;
    const bool row = at < rows;
    const bf16_t* qp = A.q + (size_t)(f.q0 + (row ? tok : 0)) * A.ldq + (size_t)(kvh * Gq + (row ? at - tok * Gq : 0)) * D + 16 * fq;
    a8_row(A, x[r], [&](int u) { return qp + u / 2 * 64 + u % 2 * 8; });
    seen[r] = min(A.causal ? f.past + tok : 0x7fffffff, kend - 1);
  }

  // chunk (16 codes) c of row r lies at place c ^ swz(r)
  auto swz = [](int row) { return D == 64 ? (row >> 1) & 3 : row & 7; };
  unsigned voff[NL / 2];
#pragma unroll
  for (int j = 0; j < NL / 2; ++j) {
    const int r = j * RPL + lane / LPR;
    voff[j] = r * D + (((lane % LPR) ^ swz(r)) * 16);
  }
  const unsigned ring = (unsigned)(size_t)(A8_LDS unsigned char*)lds + wave * L::RING;
  // A tile's loads (as many, where it has none, that reach nothing: the wait counts stay the same), 16 rows at a time, which a
  // page holds whole. The scales: lanes 0, 1 of the keys' two pages, 2, 3 of the values'.
  auto ask = [&](int kt, unsigned slot, int p0, int p1) __attribute__((always_inline)) {
    const int n = min(max(kend - kt, 0), A8_TILE);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int at = kt + 16 * t, page = t ? p1 : p0;
      const bool there = (unsigned)page < (unsigned)A.n_blocks;
      const size_t off = ((((size_t)(there ? page : 0) * A.G + kvh) << A.sh) + (at & ((1 << A.sh) - 1))) * D;
      const unsigned bytes = there ? min(max(n - 16 * t, 0), 16) * D : 0;
      const a8_u4 rk = a8_raw(A.k + off, bytes), rv = a8_raw(A.v + off, bytes);
#pragma unroll
      for (int j = 0; j < NL / 2; ++j) {
        a8_load16(rk, voff[j], slot + (t * (NL / 2) + j) * 1024);
        a8_load16(rv, voff[j], slot + L::TB + (t * (NL / 2) + j) * 1024);
      }
    }
    const int p = lane & 1 ? p1 : p0;
    a8_load4((lane & 2 ? A.vs : A.ks) + ((unsigned)p < (unsigned)A.n_blocks ? (size_t)p * A.G + kvh : 0), slot + 2 * L::TB);
  };
  constexpr int LOADS = 2 * NL + 1;
  static_assert(NL >= 2 && NL % 2 == 0, "whole loads of 16 rows");
  ask(kt0, ring, pa0, pa1);
  if constexpr (R > 1) ask(kt0 + STEP, ring + L::STAGE, pb0, pb1);

  // (waits for the rows, and with them for the tiles behind, which the compiler does not count)
  c8_h8 qf[RT][2 * NS];
  float factor[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int e = a8_lift(a8_max16(fl_max32(a8_top(x[r]))));
    factor[r] = ldexpf(A.scale_log2, -e);
    a8_queries(x[r], 16 * r + li < rows, e, false, qf[r]);
  }
  unsigned kat[NS], vat[ND];                     // places of the fragments in a stage
#pragma unroll
  for (int s = 0; s < NS; ++s) kat[s] = ring + li * D + (((4 * s + fq) ^ swz(li)) * 16);
  // lane i of 16 names row i / 2 of its eight (keys 4 fq .. + 3 of both halves), bytes 8 (i % 2) ..; it gets column i
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const int r = 16 * (li >> 3) + 4 * fq + ((li >> 1) & 3);
    vat[d] = ring + L::TB + r * D + ((d ^ swz(r)) * 16) + (li & 1) * 8;
  }
  float4v acc[RT][ND];
  float m_run[RT], l_run[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[r][d] = float4v{0.f, 0.f, 0.f, 0.f};
    m_run[r] = A8_NONE;
    l_run[r] = 0.f;
  }
  unsigned slot = 0;
  for (int kt = kt0; kt < kend; kt += STEP) {
    int next0 = 0, next1 = 0;                    // wanted behind this tile's work
    if constexpr (R > 1) { next0 = page_at(kt + 2 * STEP); next1 = page_at(kt + 2 * STEP + 16); }
    a8_wait<(R - 1) * LOADS>();                  // this tile is here, the next one's loads may be under way
    const float4v sc = *a8_lds<float4v>(ring + slot + 2 * L::TB);
    c8_u4 kw[2 * NS];
#pragma unroll
    for (int u = 0; u < 2 * NS; ++u) kw[u] = *a8_lds<c8_u4>(kat[u >> 1] + slot + 16 * (u & 1) * D);
    a8_v2i vw[ND];                               // asked for here, wanted behind the exponentials
#pragma unroll
    for (int d = 0; d < ND; ++d) vw[d] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(a8_lds<a8_v2i>(vat[d] + slot));
    float4v st[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r) st[r][0] = st[r][1] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < 2 * NS; ++u) {
      const c8_h8 lo = c8_widen8<KIND>(kw[u][0], kw[u][1]), hi = c8_widen8<KIND>(kw[u][2], kw[u][3]);
#pragma unroll
      for (int r = 0; r < RT; ++r) st[r][u & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, qf[r][u & ~1], st[r][u & 1], 0, 0, 0);
#pragma unroll
      for (int r = 0; r < RT; ++r) st[r][u & 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, qf[r][u | 1], st[r][u & 1], 0, 0, 0);
    }
    float ks[2], lv[2], inv[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool there = (unsigned)(t ? pa1 : pa0) < (unsigned)A.n_blocks;
      const float vs = c8_least(sc[2 + t]);
      ks[t] = there ? c8_least(sc[t]) : 0.f;
      lv[t] = there ? __builtin_amdgcn_logf(vs) : -INFINITY;
      inv[t] = there ? __builtin_amdgcn_rcpf(vs) * A8_DOWN : 0.f;
    }
    const bool edge = kt + A8_TILE > kend || (A.causal && kt + A8_TILE - 1 > f.past);
    c8_h8 p[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float c = factor[r] * ks[t];
#pragma unroll
        for (int j = 0; j < 4; ++j) st[r][t][j] = fmaf(st[r][t][j], c, lv[t]);
      }
      float per[2] = {inv[0], inv[1]};           // of a page that the row sees no key of (it may be another sequence's, its scale no number): 0
      if (edge) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (kt + 16 * t > seen[r]) per[t] = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (kt + 16 * t + 4 * fq + j > seen[r]) st[r][t][j] = -INFINITY;
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) mx = fmaxf(mx, st[r][j >> 2][j & 3]);
      mx = a8_max16(fl_max32(mx));
      if (__any(mx - m_run[r] > A8_MOST)) {      // as in the prompt form; the difference is what the weights have
        const float m_new = fmaxf(m_run[r], mx - A8_BELOW), alpha = __builtin_amdgcn_exp2f(m_run[r] - m_new);
        m_run[r] = m_new;
        l_run[r] *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[r][d][j] *= alpha;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float e = __builtin_amdgcn_exp2f(st[r][t][j] - m_run[r]);
          sum += e;
          p[r][4 * t + j] = (_Float16)e;
        }
        l_run[r] = fmaf(sum, per[t], l_run[r]);  // of this lane's keys
      }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const c8_h8 w = c8_widen8<KIND>(vw[d][0], vw[d][1]);
#pragma unroll
      for (int r = 0; r < RT; ++r) acc[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, p[r], acc[r][d], 0, 0, 0);
    }
    if constexpr (R > 1) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the slot has been read
      ask(kt + 2 * STEP, ring + slot, next0, next1);
      pa0 = pb0; pa1 = pb1; pb0 = next0; pb1 = next1;
      slot = slot ? 0 : L::STAGE;
    } else if (kt + STEP < kend) {               // only where a context is longer than the bound that the host gave
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      pa0 = page_at(kt + STEP); pa1 = page_at(kt + STEP + 16);
      ask(kt + STEP, ring, pa0, pa1);
    }
  }
  a8_wait<0>();                                  // no load into LDS outlives the loop
  __syncthreads();
  float* so = reinterpret_cast<float*>(lds);             // [wave][row][LD]
  float* sm = so + A8_WAVES * ROWS * LD;                 // [wave][m, l][row]
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int at = 16 * r + li;
    const float l = a8_sum16(fl_both32(l_run[r]));
    if (at >= rows) continue;
#pragma unroll
    for (int d = 0; d < ND; ++d) *reinterpret_cast<float4v*>(so + (wave * ROWS + at) * LD + 16 * d + 4 * fq) = acc[r][d];
    if (fq == 0) {
      sm[(2 * wave) * ROWS + at] = m_run[r];
      sm[(2 * wave + 1) * ROWS + at] = l;
    }
  }
  __syncthreads();
  const size_t unit = (size_t)b * A.G + kvh;
  const bool whole = (((size_t)A.out | (size_t)A.ldo * 2) & 7) == 0;
  auto put = [&](int r, int c, const float4v& o, float l) {
    const int t = r / Gq;
    a8_put(A.out + (size_t)(f.q0 + t) * A.ldo + (size_t)(kvh * Gq + r - t * Gq) * D + c, o, l, whole);
  };
  const auto rs = a8_rsrc(A, nparts > 1 ? unit : 0, nparts > 1 ? part : 0, ROWS, D);
  for (int id = tid; id < rows * (D / 4); id += A8_WAVES * 64) {
    const int r = id / (D / 4), c = id % (D / 4) * 4;
    float ms = sm[r];
#pragma unroll
    for (int w = 1; w < A8_WAVES; ++w) ms = fmaxf(ms, sm[2 * w * ROWS + r]);
    float l = 0.f;
    float4v o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < A8_WAVES; ++w) {
      const float x = exp2f(sm[2 * w * ROWS + r] - ms);
      l += sm[(2 * w + 1) * ROWS + r] * x;
      const float4v v = *reinterpret_cast<const float4v*>(so + (w * ROWS + r) * LD + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += x * v[j];
    }
    if (nparts == 1) {
      put(r, c, o, l);
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(a8_u4, o), rs, (r * D + c) * 4, 0, 16);
      if (c == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(a8_u2, make_float2(ms, l)), rs, (ROWS * D + 2 * r) * 4, 0, 16);
    }
  }
  if (nparts == 1) return;
  if (!a8_last(A.tickets + unit * TICKET, nparts, reinterpret_cast<int*>(lds + L::MERGE - 16))) return;
  a8_join<D, ROWS, A8_WAVES * 64>(A, unit, nparts, rows, reinterpret_cast<float*>(lds), put);
}

// ------------------------------------------------------------------ prompts
// 128 rows a workgroup, 32 a wave, over tiles of 64 keys: the workgroup fetches a tile's codes to registers while it works
// on the tile before, widens them to f16 rows in LDS (two stages), and computes S^T = K Q^T and O^T += V^T P^T with
// 32 x 32 x 16 MFMAs as the bf16 form does (flash_pipe.h: layouts and swizzles). Widening rides between the scores' MFMAs, a
// group's exponentials between the MFMAs of the group before.
// What bounds it: at 128 columns two waves share a SIMD (registers, and 64 KB of stages), and of 2400 cycles that a tile of one takes
// there its vector instructions have 1500 (310 of them, 32 exponentials among them, 40 to 90 to widen its share of the codes),
// its 32 MFMAs 1024, LDS 1100; a third of a wave's time is waiting to issue, a quarter for LDS and at the barrier.
// 2048 causal rows x 32 query heads over 8 of 128 columns 58 us (0.59 PFLOP/s; the bf16 form,
// whose keys and values go to LDS as they are, 56), 1024 28, 512 18; 3 x 113 rows behind 5000 keys, 64 columns, 34.
// Taken back: pages and addresses on the scalar unit (fewer vector instructions, but a chain of scalar ones in their place: 58 -> 66 us);
// the longest parts first, counted by a lane for each block (2048 rows 79); six and eight fragments of K in flight, halves of a chunk
// swapped against bank conflicts of the writes (nothing); a wave's priority raised for products or for weights, the maxima in 16
// instructions fewer, the first weights pinned beside the second scores (nothing, 1 % at most); a long and a short block one behind the
// other in a workgroup (57); 64 rows a wave, half the reads of LDS (64 columns: no faster; 128 do not fit the registers).
#define A8P_ROWS 128
#define A8P_KEYS 64
#define A8P_PARTS 32

template <int D> struct A8Prompt {
  static constexpr int K = A8P_KEYS * D * 2, STAGE = 2 * K;
  static constexpr int SCALES = 2 * STAGE, SMEM = 2 * STAGE + 2 * 64;    // [stage][ks 4, log2 vs 4, 1 / vs 4]
};

template <int D, int KIND>
__global__ __launch_bounds__(256, 2) void attn8_prompt_kernel(Attn8Args A) {
  using L = A8Prompt<D>;
  constexpr int NS = D / 16, NDT = D / 32, CH = D / 16, N = A8P_KEYS * CH / 256;    // chunks of 16 codes a row, a thread
  static_assert(N * 256 == A8P_KEYS * CH, "whole chunks a thread");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[L::SMEM];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, li = lane & 15;
  // (sequence, kv head) from the workgroup's number modulo as many, so that a head's workgroups share an XCD's L2 where these are a
  // multiple of eight
  const int b = blockIdx.x / A.G % A.B, kvh = blockIdx.x % A.G, Gq = A.H / A.G, rank = blockIdx.x / A.G / A.B;
  const A8Feed f = a8_feed(A, b);
  // keys that some row of a block sees, in parts of whole tiles
  auto rows_of = [&](int block) { return min(f.n * Gq - block * A8P_ROWS, A8P_ROWS); };
  auto tiles_of = [&](int block) {
    const int seen = A.causal ? min(f.keys, max(f.past + (block * A8P_ROWS + rows_of(block) - 1) / Gq + 1, 0)) : f.keys;
    return (seen + A8P_KEYS - 1) / A8P_KEYS;
  };
  auto parts_of = [&](int tiles) { return min(max((tiles + A.each - 1) / A.each, 1), A.parts); };
  // blocks from the longest down; but where all of them are on the chip at once, two a compute unit, the second half from
  // the shortest up, so that a long and a short one share it
  const int turn = rank / A.parts, part = rank % A.parts;
  const int block = A.fold && turn >= (A.row_blocks + 1) / 2 ? turn - (A.row_blocks + 1) / 2 : A.row_blocks - 1 - turn;
  const int r0 = block * A8P_ROWS, rows = rows_of(block);
  if (rows <= 0) return;
  const int tiles = tiles_of(block), nparts = parts_of(tiles);
  if (part >= nparts) return;
  const int i0 = (int)((long long)tiles * part / nparts), n = (int)((long long)tiles * (part + 1) / nparts) - i0;
  const unsigned base = fl_lds_at(lds);
  const int* bt = A.bt + (size_t)b * A.max_blocks;

  // this thread's chunks: row tid / CH + i 256 / CH of the tile. Codes are asked for a tile ahead and their pages' numbers two, so
  // that no load waits for another one.
  const int cr = tid / CH, cc = tid % CH, last = max(f.keys - 1, 0), mask = (1 << A.sh) - 1;
  const unsigned page_bytes = ((unsigned)A.G << A.sh) * D;
  const unsigned char* kat = A.k + ((size_t)kvh << A.sh) * D + cc * 16;
  const long long to_v = A.v - A.k;
  uint4 kw[N], vw[N];
  int pages[N], group_page = 0;
  float sk = 0.f, sv = 0.f;
  bool there = false;
  auto look = [&](int kt) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < N; ++i) pages[i] = bt[(unsigned)min(kt + cr + i * (256 / CH), last) >> A.sh];
    group_page = bt[(unsigned)min(kt + 16 * (tid & 3), last) >> A.sh];
  };
  bool none = false;
  auto ask = [&](int kt) __attribute__((always_inline)) {
    none = kt + A8P_KEYS > last + 1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const unsigned key = min(kt + cr + i * (256 / CH), last), page = (unsigned)pages[i] < (unsigned)A.n_blocks ? pages[i] : 0;
      const unsigned char* at = kat + ((unsigned long long)page * page_bytes + (unsigned)(key & mask) * D);
      kw[i] = *reinterpret_cast<const uint4*>(at);
      vw[i] = *reinterpret_cast<const uint4*>(at + to_v);
      none |= page != (unsigned)pages[i];
    }
  };
  auto asked = [&](int kt) __attribute__((always_inline)) {    // what of it branches, and the pages of the tile behind
    if (__any(none)) {                                       // codes that are none may be NaN, which no weight of zero hides
#pragma unroll
      for (int i = 0; i < N; ++i)
        if ((unsigned)pages[i] >= (unsigned)A.n_blocks || kt + cr + i * (256 / CH) > last) kw[i] = vw[i] = make_uint4(0, 0, 0, 0);
    }
    if (tid < 4) {                                           // the scales of 16 keys
      there = (unsigned)group_page < (unsigned)A.n_blocks;
      const size_t at = (size_t)(there ? group_page : 0) * A.G + kvh;
      sk = A.ks[at];
      sv = A.vs[at];
    }
    look(kt + A8P_KEYS);
  };
  // piece q of the tile in registers: 8 codes, of keys or of values, widened and put where the fragments are read from
  constexpr int PIECES = 4 * N;
  unsigned put_at[4];                                        // K's and V's two parts in the first stage; rows further on keep the swizzle
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int sw = q & 2 ? fl_vswz<D>(cr) : fl_kswz<D>(cr);
    put_at[q] = base + (q & 2 ? L::K : 0) + cr * (D * 2) + ((2 * cc + (q & 1)) ^ sw) * 16;
  }
  auto store = [&](int stage, int q) __attribute__((always_inline)) {
    const uint4 w = q & 2 ? vw[q >> 2] : kw[q >> 2];
    *fl_lds<c8_h8>(put_at[q & 3] + stage * L::STAGE + (q >> 2) * (256 / CH) * D * 2) = q & 1 ? c8_widen8<KIND>(w.z, w.w) : c8_widen8<KIND>(w.x, w.y);
  };
  static_assert(256 / CH % 16 == 0, "a thread's rows share a swizzle");
  auto store_scales = [&](int stage) __attribute__((always_inline)) {
    if (tid < 4) {
      float* s = reinterpret_cast<float*>(lds + L::SCALES + stage * 64) + tid;
      const float vs = c8_least(sv);
      s[0] = there ? c8_least(sk) : 1.f;
      s[4] = there ? __builtin_amdgcn_logf(vs) : -INFINITY;
      s[8] = there ? __builtin_amdgcn_rcpf(vs) * A8_DOWN : 0.f;        // off by 2^-23
    }
  };

  unsigned kb[NS], vb[NDT];
#pragma unroll
  for (int s = 0; s < NS; ++s) kb[s] = base + (lane & 31) * (D * 2) + ((2 * s + h) ^ fl_kswz<D>(lane & 31)) * 16;
#pragma unroll
  for (int d = 0; d < NDT; ++d)
    vb[d] = base + L::K + (4 * h + (li >> 2)) * (D * 2) + ((4 * d + 2 * ((lane >> 4) & 1) + ((li & 3) >> 1)) ^ fl_vswz<D>(li >> 2)) * 16 + (li & 1) * 8;

  const float16v zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float16v acc[NDT];
#pragma unroll
  for (int d = 0; d < NDT; ++d) acc[d] = zero;
  float m = A8_NONE, l = 0.f;
  if (n > 0) look(i0 * A8P_KEYS);
  const int r = r0 + wave * 32 + (lane & 31), tok = min(r / Gq, f.n - 1), seen = min(A.causal ? f.past + r / Gq : 0x7fffffff, f.keys - 1);
  c8_h8 qf[NS];
  float factor;
  {
    const bool row = r < r0 + rows;
    const bf16_t* qp = A.q + (size_t)(f.q0 + tok) * A.ldq + (size_t)(kvh * Gq + r % Gq) * D + 8 * h;
    uint4 x[NS];
    a8_row(A, x, [&](int u) { return qp + 16 * u; });
    const int e = a8_lift(fl_max32(a8_top(x)));
    factor = ldexpf(fabsf(A.scale_log2), -e);                // above zero, so that a group's largest product is its largest score
    a8_queries(x, row, e, A.scale_log2 < 0.f, qf);
  }

  if (n > 0) {
    const int kt = i0 * A8P_KEYS;
    ask(kt);
    asked(kt);
#pragma unroll
    for (int q = 0; q < PIECES; ++q) store(0, q);
    store_scales(0);
    ask(kt + A8P_KEYS);
    asked(kt + A8P_KEYS);
  }
  // A tile: the scores of its first 32 keys, beside which the next tile is widened; those of the second 32; the maxima, which move the
  // reference where they have to, and the weights of the first keys; the values' products of these beside the weights of the second;
  // those of the second beside the addresses of the tile after the next. (One after the other, stages toggled in registers: the 2048
  // rows above 58 us, 56 so; the first weights beside the second scores, and once more where the reference moves: no faster.)
  constexpr int KR = 4, VR = 4;                              // fragments in flight + 1
  // rows of this wave that some key of a tile from here on is hidden from, or that end in it
  const int edge = min(f.keys, A.causal ? f.past + (r0 + wave * 32) / Gq + 1 : f.keys) - A8P_KEYS;
  auto tile = [&](auto slot, int i) __attribute__((always_inline)) {
    constexpr int stage = decltype(slot)::value;
    const int kt = (i0 + i) * A8P_KEYS;
    fl_meet();                                               // this stage is written, nobody reads the other one any more; loads stay under way
    const float* sc = reinterpret_cast<const float*>(lds + L::SCALES + stage * 64);
    const float4v ks = *reinterpret_cast<const float4v*>(sc);
    float4v lv = *reinterpret_cast<const float4v*>(sc + 4), inv = *reinterpret_cast<const float4v*>(sc + 8);
    float16v s[2];
    c8_h8 kf[KR], vf[VR], p[4];
    float sum[4], c[4], top[4], off[4];
    auto kread = [&](int u) __attribute__((always_inline)) { kf[u % KR] = *fl_lds<c8_h8>(kb[u % NS] + (stage * L::STAGE + 32 * (u / NS) * D * 2)); };
    auto vread = [&](int v) __attribute__((always_inline)) {
      const unsigned a = vb[v % NDT] + (stage * L::STAGE + 16 * (v / NDT) * D * 2);
      const fl_v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(fl_lds<fl_v4s>(a));
      const fl_v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(fl_lds<fl_v4s>(a + 8 * D * 2));
      short8 a8;
#pragma unroll
      for (int j = 0; j < 4; ++j) { a8[j] = lo[j]; a8[4 + j] = hi[j]; }
      vf[v % VR] = __builtin_bit_cast(c8_h8, a8);
    };
    auto hide = [&](int t) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (kt + 32 * t + (j & 3) + 8 * (j >> 2) + 4 * h > seen) s[t][j] = -INFINITY;
    };
    // scores j of group g (16 keys of a page): 2^(x c + log2 vs - m)
    auto weights = [&](int g, int j0, int j1) __attribute__((always_inline)) {
#pragma unroll
      for (int j = j0; j < j1; j += 2) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        const f2 e = {__builtin_amdgcn_exp2f(fmaf(s[g >> 1][8 * (g & 1) + j], c[g], off[g])),
                      __builtin_amdgcn_exp2f(fmaf(s[g >> 1][8 * (g & 1) + j + 1], c[g], off[g]))};
        const c8_h2 w = __builtin_convertvector(e, c8_h2);
        sum[g] = j == 0 ? e[0] + e[1] : sum[g] + (e[0] + e[1]);    // in f32: a weight that f16 has as zero still counts for a page of small values
        p[g][j] = w[0];
        p[g][j + 1] = w[1];
      }
    };
    auto tops = [&](int g, int j0, int j1) __attribute__((always_inline)) {
#pragma unroll
      for (int j = j0; j < j1; j += 2)
        top[g] = j == 0 ? fmaxf(s[g >> 1][8 * (g & 1)], s[g >> 1][8 * (g & 1) + 1])
                        : fmaxf(fmaxf(top[g], s[g >> 1][8 * (g & 1) + j]), s[g >> 1][8 * (g & 1) + j + 1]);
    };
#pragma unroll
    for (int u = 0; u < KR - 1; ++u) kread(u);
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[u % KR], qf[u], u == 0 ? zero : s[0], 0, 0, 0);
      kread(u + KR - 1);
      store(1 - stage, u);
      __builtin_amdgcn_sched_barrier(0);
    }
    static_assert(PIECES == NS && KR - 1 <= NS, "a piece for every MFMA");
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float k = factor * ks[g];
      c[g] = k < 1.1754943508222875e-38f ? 1.1754943508222875e-38f : k;     // of no use to a masked -infinity if zero; NaN stays
    }
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[(NS + u) % KR], qf[u], u == 0 ? zero : s[1], 0, 0, 0);
      if (u + KR - 1 < NS) kread(NS + u + KR - 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    store_scales(1 - stage);
#pragma unroll
    for (int v = 0; v < VR - 1; ++v) vread(v);
    if (kt > edge) {
      hide(0);
      hide(1);
#pragma unroll
      for (int g = 0; g < 4; ++g)
        if (kt + 16 * g > seen) {                            // keys that the row sees none of: their page's scales, which may be no numbers, are not its own
          c[g] = 1.f;
          lv[g] = -INFINITY;
          inv[g] = 0.f;
        }
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) tops(g, 0, 8);
    // x c + log2 vs with c above zero: the largest product of a group is its largest score. The reference stays where it is while no
    // weight passes 2^15, up to which f16 keeps 11 bits (a prompt's first tiles nearly always raise some row of the wave): asked of the
    // weights' own exponents, as scores past 2^23 have steps that a sum of 15 would be rounded to
    float mx = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      off[g] = lv[g] - m;
      mx = fmaxf(mx, fmaf(top[g], c[g], off[g]));
    }
    if (__any(mx > A8_MOST)) {
      mx = -INFINITY;
#pragma unroll
      for (int g = 0; g < 4; ++g) mx = fmaxf(mx, fmaf(top[g], c[g], lv[g]));
      mx = fl_max32(mx);
      const float m_new = fmaxf(m, mx - A8_BELOW), alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < NDT; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[d][j] *= alpha;
#pragma unroll
      for (int g = 0; g < 4; ++g) off[g] = lv[g] - m;
    }
    weights(0, 0, 8);
    weights(1, 0, 8);
    __builtin_amdgcn_sched_barrier(0);
    constexpr int PW = 16 / (2 * NDT);
#pragma unroll
    for (int v = 0; v < 2 * NDT; ++v) {
      acc[v % NDT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[v % VR], p[v / NDT], acc[v % NDT], 0, 0, 0);
      vread(v + VR - 1);
      weights(2 + v * PW / 8, v * PW % 8, v * PW % 8 + PW);
      __builtin_amdgcn_sched_barrier(0);
    }
    ask(kt + 2 * A8P_KEYS);
#pragma unroll
    for (int v = 2 * NDT; v < 4 * NDT; ++v) {
      acc[v % NDT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[v % VR], p[v / NDT], acc[v % NDT], 0, 0, 0);
      if (v + VR - 1 < 4 * NDT) vread(v + VR - 1);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) l = fmaf(sum[g], inv[g], l);
    asked(kt + 2 * A8P_KEYS);
  };
  for (int i = 0; i < n; i += 2) {                           // a stage's places are constants of its copy of the code
    tile(Fl<0>{}, i);
    if (i + 1 < n) tile(Fl<1>{}, i + 1);
  }
  l = fl_both32(l);                                          // a lane has summed up its half of the keys
  const size_t unit = ((size_t)b * A.G + kvh) * A.row_blocks + block;
  const bool whole = (((size_t)A.out | (size_t)A.ldo * 2) & 7) == 0;
  const int row = wave * 32 + (lane & 31);
  // Parts of a block's keys: each leaves its accumulators as they lie (16 bytes a lane, a kilobyte a wave), and the last to arrive
  // adds up all of them, in order.
  if (nparts > 1) {
    constexpr int PER = 256 * (NDT * 16 + 2) * 4;
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(A.ws + unit * A.parts * (PER / 4), 0, A.parts * PER, 0x00020000);
    const int at = part * PER + tid * 16, ml = 256 * NDT * 16 * 4 + tid * 8;
    const bool some = wave * 32 < rows;                      // a wave without rows leaves nothing
    if (some) {
#pragma unroll
      for (int u = 0; u < 4 * NDT; ++u) {
        const float4v o = {acc[u / 4][u % 4 * 4], acc[u / 4][u % 4 * 4 + 1], acc[u / 4][u % 4 * 4 + 2], acc[u / 4][u % 4 * 4 + 3]};
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(a8_u4, o), rs, at + u * 4096, 0, 16);
      }
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(a8_u2, make_float2(m, l)), rs, part * PER + ml, 0, 16);
    }
    if (!a8_last(A.tickets + unit * TICKET, nparts, reinterpret_cast<int*>(lds)) || !some) return;
    float top = A8_NONE, all = 0.f;
    float tops[A8P_PARTS];                                   // all asked for together
#pragma unroll
    for (int p = 0; p < A8P_PARTS; ++p) tops[p] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rs, min(p, nparts - 1) * PER + ml, 0, 16));
#pragma unroll
    for (int p = 0; p < A8P_PARTS; ++p) top = fmaxf(top, tops[p]);
#pragma unroll
    for (int d = 0; d < NDT; ++d) acc[d] = zero;
    constexpr int GP = 8 / NDT;                              // parts under way together
    for (int p0 = 0; p0 < nparts; p0 += GP) {
      float4v v[GP][4 * NDT];
      float2 w[GP];
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        const int p = min(p0 + g, nparts - 1);
        w[g] = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(rs, p * PER + ml, 0, 16));
#pragma unroll
        for (int u = 0; u < 4 * NDT; ++u) v[g][u] = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(rs, p * PER + tid * 16 + u * 4096, 0, 16));
      }
#pragma unroll
      for (int g = 0; g < GP; ++g) {
        if (p0 + g >= nparts) break;
        const float x = __builtin_amdgcn_exp2f(w[g].x - top);
        all = fmaf(x, w[g].y, all);
#pragma unroll
        for (int u = 0; u < 4 * NDT; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[u / 4][u % 4 * 4 + j] = fmaf(x, v[g][u][j], acc[u / 4][u % 4 * 4 + j]);
      }
    }
    l = all;
  }
  if (row < rows) {
    const int t = (r0 + row) / Gq;
    bf16_t* at = A.out + (size_t)(f.q0 + t) * A.ldo + (size_t)(kvh * Gq + r0 + row - t * Gq) * D + 4 * h;
    const float by = l == 0.f ? 0.f : 1.f / l;               // NaN stays
#pragma unroll
    for (int u = 0; u < 4 * NDT; ++u) {                      // accumulators 4 u ..: columns 8 u + 4 h ..
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = acc[u / 4][u % 4 * 4 + j] * A8_DOWN * by;
      const uint2 w = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
      if (whole) {
        *reinterpret_cast<uint2*>(at + 8 * u) = w;
      } else {
        at[8 * u] = (bf16_t)w.x; at[8 * u + 1] = (bf16_t)(w.x >> 16); at[8 * u + 2] = (bf16_t)w.y; at[8 * u + 3] = (bf16_t)(w.y >> 16);
      }
    }
  }
}

// form: 0 prompts, 1 or 2 token steps of up to 16 times as many rows; parts: of a sequence's keys at most; each: tiles of 64 keys of a
// prompt's part (the longer blocks have more parts); of a token step 1 where a wave is expected to have one tile (parts * 128 keys bound
// the contexts), else 2
extern "C" int loqa_attention8(const void* q, long ldq, const void* k, const void* v, const void* ks, const void* vs, const void* cu,
                               const void* ctx, const void* bt, void* out, long ldo, int T, int B, int H, int G, int D, int blk, int n_blocks,
                               int max_blocks, int max_q, float scale, int causal, int kind, int form, int parts, int each, void* ws, long ws_floats, void* tickets,
                               long n_tickets, hipStream_t st) {
  if (T <= 0 || B <= 0 || max_q <= 0) return 0;
  if ((D != 64 && D != 128) || (kind != C8_INT8 && kind != C8_E4M3) || blk < 16 || (blk & (blk - 1)) || G <= 0 || H <= 0 || H % G ||
      n_blocks <= 0 || max_blocks <= 0 || parts <= 0 || each <= 0)
    return (int)hipErrorInvalidValue;
  const bool token = form > 0;
  if (form < 0 || form > 2 || (token && (long long)max_q * (H / G) > 16 * form)) return (int)hipErrorInvalidValue;
  const long long blocks = token ? 1 : ((long long)max_q * (H / G) + A8P_ROWS - 1) / A8P_ROWS, units = (long long)B * G * blocks;
  const long long per = token ? 16 * form * (D + 2) : A8P_ROWS * (D + 4);     // floats of a part
  if (!token && parts > A8P_PARTS) return (int)hipErrorInvalidValue;
  if (token ? G > 65535 || B > 65535 || parts > 1 << 24 : units * parts > 1 << 30) return (int)hipErrorInvalidValue;
  if ((long long)G * blk * D >= 1LL << 31 || blocks > 1 << 24 || parts * per * 4 >= 1LL << 31)
    return (int)hipErrorInvalidValue;
  if (parts > 1 && (!ws || !tickets || ws_floats < units * parts * per || n_tickets < units)) return (int)hipErrorInvalidValue;
  const Attn8Args a{(const bf16_t*)q, ldq, (const unsigned char*)k, (const unsigned char*)v, (const float*)ks, (const float*)vs, (const int*)cu,
                    (const int*)ctx, (const int*)bt, (bf16_t*)out, ldo, (float*)ws, (int*)tickets, T, B, H, G, __builtin_ctz(blk), n_blocks, max_blocks,
                    max_q, parts, causal, (int)blocks, each, parts == 1 && units <= 512, scale * 1.4426950408889634f};
  if (token) {
    const dim3 grid(parts, G, B);
#define GO1(D_, K_, R_, RT_) hipLaunchKernelGGL((attn8_token_kernel<D_, K_, R_, RT_>), grid, dim3(A8_WAVES * 64), 0, st, a)
#define GO(D_, K_) do { if (form == 2) { if (each == 1) GO1(D_, K_, 1, 2); else GO1(D_, K_, 2, 2); } \
                        else if (each == 1) GO1(D_, K_, 1, 1); else GO1(D_, K_, 2, 1); } while (0)
    if (D == 64) { if (kind == C8_INT8) GO(64, C8_INT8); else GO(64, C8_E4M3); }
    else { if (kind == C8_INT8) GO(128, C8_INT8); else GO(128, C8_E4M3); }
#undef GO
#undef GO1
  } else {
    const dim3 grid((unsigned)(units * parts));
#define GO(D_, K_) hipLaunchKernelGGL((attn8_prompt_kernel<D_, K_>), grid, dim3(256), 0, st, a)
    if (D == 64) { if (kind == C8_INT8) GO(64, C8_INT8); else GO(64, C8_E4M3); }
    else { if (kind == C8_INT8) GO(128, C8_INT8); else GO(128, C8_E4M3); }
#undef GO
  }
  return (int)hipGetLastError();
}
