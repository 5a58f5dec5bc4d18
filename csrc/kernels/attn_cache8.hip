// Attention off the paged cache in 8 bits (cache8.h). Rows r of a feed are its tokens times the G query heads of a kv
// head, token r / G and head r % G: every key and value is read, and widened to f16, once for all of them.
//
//   x_j = q . k_j (f16 MFMAs, f32 sums),  s_j = scale log2(e) ks x_j,  o = sum_j 2^(s_j) vs v_j / sum_j 2^(s_j)
//
// with ks, vs of a key's page. The values' scale goes into the exponent: t_j = s_j + log2(vs), weights w_j = 2^(t_j - max t)
// are what the codes of v are summed up with, at most one and so f16 without a range of their own (11 bits; under 2^-14
// an absolute 2^-25), and the denominator is sum_j w_j / vs in f32. Queries enter as f16 times a power of two of
// the row that puts its largest entry in 2^14 .. 2^15: bf16's 8 bits are exact down to 2^-28 of it.
//
// Rows that see no key (a position before the first) give zeros; keys of pages that do not exist count as masked.
#include "cache8.h"
#include "flash_pipe.h"

#define A8_NONE -3.0e38f                           // a row's maximum before its first key

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
  int T, B, H, G, sh, n_blocks, max_blocks, max_q, parts, causal, row_blocks, fold;
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

__device__ __forceinline__ float a8_least(float s) { return s < C8_LEAST ? C8_LEAST : s; }   // NaN stays

// eight entries of a query row in f32 (bf16 at any 2-byte place), zeros for a row that is none
__device__ __forceinline__ void a8_row8(const bf16_t* p, bool whole, float* f) {
  if (whole) {
    unpack8(*reinterpret_cast<const uint4*>(p), f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = bf2f(p[i]);
  }
}

// the power of two that puts a largest magnitude into 2^14 .. 2^15, as an exponent (0 for a row of zeros)
__device__ __forceinline__ int a8_lift(float top) {
  return top > 0.f && top < INFINITY ? min(14 - (int)((__float_as_uint(top) >> 23) & 255) + 127, 126) : 0;
}

// ---- the partials of a row block's parts, joined by the last of them. R rows; a thread's accumulators are put at
// (row, column), four columns a piece. Written through and read past the caches: parts may run on different XCDs.
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
  const uint2 w = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
  if (whole) {
    *reinterpret_cast<uint2*>(at) = w;
  } else {
    at[0] = (bf16_t)w.x; at[1] = (bf16_t)(w.x >> 16); at[2] = (bf16_t)w.y; at[3] = (bf16_t)(w.y >> 16);
  }
}

// joins n parts of `rows` rows in order and writes them; NT threads, eight partials under way
template <int D, int R, int NT, typename Put>
__device__ __forceinline__ void a8_join(const Attn8Args& A, size_t unit, int n, int rows, Put&& put) {
  constexpr int OB = 8, PER = R * (D + 2) * 4;
  const auto rs = __builtin_amdgcn_make_buffer_rsrc(A.ws + unit * A.parts * R * (D + 2), 0, A.parts * PER, 0x00020000);
  for (int id = threadIdx.x; id < rows * (D / 4); id += NT) {
    const int r = id / (D / 4), c = id % (D / 4) * 4;
    float ms = A8_NONE, l = 0.f;
    float4v o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < n; s0 += OB) {
      float4v v[OB];
      float2 ml[OB];
#pragma unroll
      for (int i = 0; i < OB; ++i) {
        const int at = min(s0 + i, n - 1) * PER;
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
        if (s0 + i >= n) break;
        const float x = exp2f(ml[i].x - ms);
        l += x * ml[i].y;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += x * v[i][j];
      }
    }
    put(r, c, o, l);
  }
}

// ------------------------------------------------------------------ token steps
// Up to 16 rows per kv head. A step reads every cached code once, so it is bound by the bytes a compute unit has
// under way: each wave streams tiles of 32 keys straight to its own ring of two in LDS, as the bf16 form does
// (attn_stream.hip), the scales of a tile's two pages with it. The waves of a workgroup take tiles in turn, the
// workgroups of a sequence parts of its keys.
//
//   S^T = K Q^T   : 16 x 16 x 32 MFMAs; a lane reads 16 codes of a key at once, the K slots of two MFMAs
//   O^T += V^T P^T: eight keys of one column by a transposing read of bytes; P^T is the accumulator as it stands
#define A8_ROWS 16
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

template <int D> struct A8Token {
  static constexpr int TB = A8_TILE * D, STAGE = 2 * TB + 256;         // K, V, a dword a lane of scales
  static constexpr int RING = 2 * STAGE;
  static constexpr int MERGE = A8_WAVES * A8_ROWS * (D + 4 + 2) * 4 + 16;
  static constexpr int SMEM = A8_WAVES * RING > MERGE ? A8_WAVES * RING : MERGE;
};

template <int D, int KIND>
__global__ __launch_bounds__(A8_WAVES * 64) void attn8_token_kernel(Attn8Args A) {
  using L = A8Token<D>;
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
  auto page_at = [&](int kt, int i) { return a8_scalar(bt + min((kt + 16 * i) >> A.sh, A.max_blocks - 1)); };

  // the queries of row li: K slots (fq, e) of MFMAs 2 s and 2 s + 1 are columns 64 s + 16 fq + e and + 8 + e
  const int tok = li / Gq;
  c8_h8 qf[2 * NS];
  float factor;
  {
    const bool row = li < rows, whole = (((size_t)A.q | (size_t)A.ldq * 2) & 15) == 0;
    const bf16_t* qp = A.q + (size_t)(f.q0 + tok) * A.ldq + (size_t)(kvh * Gq + li - tok * Gq) * D + 16 * fq;
    float x[2 * NS][8];
    float top = 0.f;
#pragma unroll
    for (int u = 0; u < 2 * NS; ++u) {
      if (row) a8_row8(qp + u / 2 * 64 + u % 2 * 8, whole, x[u]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!row) x[u][i] = 0.f;
        top = fmaxf(top, fabsf(x[u][i]));
      }
    }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const int e = a8_lift(top);
    factor = ldexpf(A.scale_log2, -e);
#pragma unroll
    for (int u = 0; u < 2 * NS; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) qf[u][i] = (_Float16)ldexpf(x[u][i], e);
#pragma unroll
    for (int u = 0; u < 2 * NS; ++u) asm volatile("" : "+v"(qf[u]));   // here before the loads whose count the compiler does not know
    asm volatile("" : "+v"(factor));
  }
  const int qpos = A.causal ? f.past + tok : 0x7fffffff;

  // chunk (16 codes) c of row r lies at place c ^ swz(r)
  auto swz = [](int row) { return D == 64 ? (row >> 1) & 3 : row & 7; };
  unsigned voff[NL];
#pragma unroll
  for (int j = 0; j < NL; ++j) {
    const int r = j * RPL + lane / LPR;
    voff[j] = (r & 15) * D + (((lane % LPR) ^ swz(r)) * 16);
  }
  const unsigned ring = (unsigned)(size_t)(A8_LDS unsigned char*)lds + wave * L::RING;
  // A tile's loads (as many, where it has none, that reach nothing: the wait counts stay the same), 16 rows at a time, which a
  // page holds whole. The scales: lanes 0, 1 of the keys' two pages, 2, 3 of the values'.
  auto ask = [&](int kt, unsigned slot, const int (&page)[2]) {
    const int n = min(max(kend - kt, 0), A8_TILE);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int at = kt + 16 * t;
      const bool there = (unsigned)page[t] < (unsigned)A.n_blocks;
      const size_t off = ((((size_t)(there ? page[t] : 0) * A.G + kvh) << A.sh) + (at & ((1 << A.sh) - 1))) * D;
      const unsigned bytes = there ? min(max(n - 16 * t, 0), 16) * D : 0;
      const a8_u4 rk = a8_raw(A.k + off, bytes), rv = a8_raw(A.v + off, bytes);
#pragma unroll
      for (int j = t * (NL / 2); j < (t + 1) * (NL / 2); ++j) {
        a8_load16(rk, voff[j], slot + j * 1024);
        a8_load16(rv, voff[j], slot + L::TB + j * 1024);
      }
    }
    const int p = lane & 1 ? page[1] : page[0];
    a8_load4((lane & 2 ? A.vs : A.ks) + ((unsigned)p < (unsigned)A.n_blocks ? (size_t)p * A.G + kvh : 0), slot + 2 * L::TB);
  };
  constexpr int LOADS = 2 * NL + 1;
  static_assert(NL >= 2 && NL % 2 == 0, "whole loads of 16 rows");

  float4v acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = float4v{0.f, 0.f, 0.f, 0.f};
  float m_run = A8_NONE, l_run = 0.f;
  int pages[2][2] = {{page_at(kt0, 0), page_at(kt0, 1)}, {page_at(kt0 + STEP, 0), page_at(kt0 + STEP, 1)}};
  ask(kt0, ring, pages[0]);
  ask(kt0 + STEP, ring + L::STAGE, pages[1]);
  unsigned slot = ring;
  for (int kt = kt0; kt < kend; kt += STEP) {
    int next[2] = {page_at(kt + 2 * STEP, 0), page_at(kt + 2 * STEP, 1)};       // wanted behind this tile's work
    a8_wait<LOADS>();                            // this tile is here, the next one's loads may be under way
    const float4v sc = *a8_lds<float4v>(slot + 2 * L::TB);
    float4v st[2] = {float4v{0.f, 0.f, 0.f, 0.f}, float4v{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const c8_u4 w = *a8_lds<c8_u4>(slot + (16 * t + li) * D + (((4 * s + fq) ^ swz(16 * t + li)) * 16));
        st[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c8_widen8<KIND>(w[0], w[1]), qf[2 * s], st[t], 0, 0, 0);
        st[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c8_widen8<KIND>(w[2], w[3]), qf[2 * s + 1], st[t], 0, 0, 0);
      }
    float mx = -INFINITY, inv[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool there = (unsigned)pages[0][t] < (unsigned)A.n_blocks;
      const float vs = a8_least(sc[2 + t]), c = there ? factor * sc[t] : 0.f, lv = there ? __builtin_amdgcn_logf(vs) : -INFINITY;
      inv[t] = there ? 1.f / vs : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = kt + 16 * t + 4 * fq + j;
        float sv = fmaf(st[t][j], c, lv);
        if (key >= kend || key > qpos) sv = -INFINITY;
        st[t][j] = sv;
        mx = fmaxf(mx, sv);
      }
    }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float m_new = fmaxf(m_run, mx), alpha = exp2f(m_run - m_new);
    m_run = m_new;
    c8_h8 p;
    float ls = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = exp2f(st[t][j] - m_new);
        sum += e;
        p[4 * t + j] = (_Float16)e;
      }
      ls = fmaf(sum, inv[t], ls);
    }
    l_run = l_run * alpha + ls;                  // of this lane's keys
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      // lane i of 16 names row i / 2 of its eight (keys 4 fq .. + 3 of both halves), bytes 8 (i % 2) ..; it gets column i
      const int row = 16 * (li >> 3) + 4 * fq + ((li >> 1) & 3);
      const a8_v2i w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(a8_lds<a8_v2i>(slot + L::TB + row * D + ((d ^ swz(row)) * 16) + (li & 1) * 8));
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[d][j] *= alpha;
      acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(c8_widen8<KIND>(w[0], w[1]), p, acc[d], 0, 0, 0);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the slot has been read
    ask(kt + 2 * STEP, slot, next);
    pages[0][0] = pages[1][0]; pages[0][1] = pages[1][1];
    pages[1][0] = next[0]; pages[1][1] = next[1];
    slot = slot == ring ? ring + L::STAGE : ring;
  }
  a8_wait<0>();                                  // no load into LDS outlives the loop
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  __syncthreads();
  float* so = reinterpret_cast<float*>(lds);             // [wave][row][LD]
  float* sm = so + A8_WAVES * A8_ROWS * LD;              // [wave][m, l][row]
  if (li < rows) {
#pragma unroll
    for (int d = 0; d < ND; ++d) *reinterpret_cast<float4v*>(so + (wave * A8_ROWS + li) * LD + 16 * d + 4 * fq) = acc[d];
    if (fq == 0) {
      sm[(2 * wave) * A8_ROWS + li] = m_run;
      sm[(2 * wave + 1) * A8_ROWS + li] = l_run;
    }
  }
  __syncthreads();
  const size_t unit = (size_t)b * A.G + kvh;
  const bool whole = (((size_t)A.out | (size_t)A.ldo * 2) & 7) == 0;
  auto put = [&](int r, int c, const float4v& o, float l) {
    const int t = r / Gq;
    a8_put(A.out + (size_t)(f.q0 + t) * A.ldo + (size_t)(kvh * Gq + r - t * Gq) * D + c, o, l, whole);
  };
  const auto rs = a8_rsrc(A, nparts > 1 ? unit : 0, nparts > 1 ? part : 0, A8_ROWS, D);
  for (int id = tid; id < rows * (D / 4); id += A8_WAVES * 64) {
    const int r = id / (D / 4), c = id % (D / 4) * 4;
    float ms = sm[r];
#pragma unroll
    for (int w = 1; w < A8_WAVES; ++w) ms = fmaxf(ms, sm[2 * w * A8_ROWS + r]);
    float l = 0.f;
    float4v o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < A8_WAVES; ++w) {
      const float x = exp2f(sm[2 * w * A8_ROWS + r] - ms);
      l += sm[(2 * w + 1) * A8_ROWS + r] * x;
      const float4v v = *reinterpret_cast<const float4v*>(so + (w * A8_ROWS + r) * LD + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += x * v[j];
    }
    if (nparts == 1) {
      put(r, c, o, l);
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(a8_u4, o), rs, (r * D + c) * 4, 0, 16);
      if (c == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(a8_u2, make_float2(ms, l)), rs, (A8_ROWS * D + 2 * r) * 4, 0, 16);
    }
  }
  if (nparts == 1) return;
  if (!a8_last(A.tickets + unit * TICKET, nparts, reinterpret_cast<int*>(lds + L::MERGE - 16))) return;
  a8_join<D, A8_ROWS, A8_WAVES * 64>(A, unit, nparts, rows, put);
}

// ------------------------------------------------------------------ prompts
// 128 rows a workgroup, 32 a wave, over tiles of 64 keys: the workgroup fetches a tile's codes to registers while it works
// on the tile before, widens them to f16 rows in LDS (two stages), and computes S^T = K Q^T and O^T += V^T P^T with
// 32 x 32 x 16 MFMAs as the bf16 form does (flash_pipe.h: layouts and swizzles).
#define A8P_ROWS 128
#define A8P_KEYS 64

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
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, li = lane & 15;
  // (sequence, kv head) from the workgroup's number modulo as many, so that a head's workgroups share an XCD's L2 where these are a
  // multiple of eight; blocks of rows from the longest down, but the second of two workgroups a compute unit from the
  // shortest up: with all of them on the chip at once, a long and a short one share it
  const int b = blockIdx.x / A.G % A.B, kvh = blockIdx.x % A.G, Gq = A.H / A.G;
  const int rest = blockIdx.x / A.G / A.B, part = rest % A.parts, turn = rest / A.parts;
  const A8Feed f = a8_feed(A, b);
  const int half = (A.row_blocks + 1) / 2;
  const int block = A.fold && turn >= half ? turn - half : A.row_blocks - 1 - turn;
  const int r0 = block * A8P_ROWS, rows = min(f.n * Gq - r0, A8P_ROWS);
  if (rows <= 0) return;
  // keys that some row of the block sees, in parts of whole tiles
  const int seen = A.causal ? min(f.keys, max(f.past + (r0 + rows - 1) / Gq + 1, 0)) : f.keys;
  const int tiles = (seen + A8P_KEYS - 1) / A8P_KEYS, each = max((tiles + A.parts - 1) / A.parts, 1);
  const int nparts = max((tiles + each - 1) / each, 1);
  if (part >= nparts) return;
  const int i0 = part * each, n = min(tiles, i0 + each) - i0;
  const unsigned base = fl_lds_at(lds);
  const int* bt = A.bt + (size_t)b * A.max_blocks;

  const int r = r0 + wave * 32 + (lane & 31), tok = min(r / Gq, f.n - 1), qpos = A.causal ? f.past + r / Gq : 0x7fffffff;
  c8_h8 qf[NS];
  float factor;
  {
    const bool row = r < r0 + rows, whole = (((size_t)A.q | (size_t)A.ldq * 2) & 15) == 0;
    const bf16_t* qp = A.q + (size_t)(f.q0 + tok) * A.ldq + (size_t)(kvh * Gq + r % Gq) * D + 8 * h;
    float top = 0.f;
    float x[NS][8];
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      if (row) a8_row8(qp + 16 * u, whole, x[u]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!row) x[u][i] = 0.f;
        top = fmaxf(top, fabsf(x[u][i]));
      }
    }
    top = fl_max32(top);
    const int e = a8_lift(top);
    factor = ldexpf(fabsf(A.scale_log2), -e);
    const float sign = A.scale_log2 < 0.f ? -1.f : 1.f;      // a factor above zero keeps a group's largest product its largest score
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) qf[u][i] = (_Float16)(sign * ldexpf(x[u][i], e));
  }

  // this thread's chunks: row tid / CH + i 256 / CH of the tile
  const int cr = tid / CH, cc = tid % CH;
  // Codes are asked for a tile ahead and their pages' numbers two, so that no load waits for another one.
  const int last = max(f.keys - 1, 0);
  uint4 kw[N], vw[N];
  int pages[N], group_page = 0;
  float sk = 0.f, sv = 0.f;
  bool there = false;
  auto look = [&](int tile) {
    const int kt = tile * A8P_KEYS;
#pragma unroll
    for (int i = 0; i < N; ++i) pages[i] = bt[min(kt + cr + i * (256 / CH), last) >> A.sh];
    group_page = bt[min(kt + 16 * (tid & 3), last) >> A.sh];
  };
  auto fetch = [&](int tile) {
    const int kt = tile * A8P_KEYS;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int key = min(kt + cr + i * (256 / CH), last);
      const bool ok = (unsigned)pages[i] < (unsigned)A.n_blocks;
      const size_t off = ((((size_t)(ok ? pages[i] : 0) * A.G + kvh) << A.sh) + (key & ((1 << A.sh) - 1))) * D + cc * 16;
      kw[i] = *reinterpret_cast<const uint4*>(A.k + off);
      vw[i] = *reinterpret_cast<const uint4*>(A.v + off);
      if (__any(!ok || kt + cr + i * (256 / CH) > last)) {   // codes that are none may be NaN, which no weight of zero hides
        if (!ok || kt + cr + i * (256 / CH) > last) kw[i] = vw[i] = make_uint4(0, 0, 0, 0);
      }
    }
    if (tid < 4) {                                           // the scales of 16 keys
      there = (unsigned)group_page < (unsigned)A.n_blocks;
      const size_t at = (size_t)(there ? group_page : 0) * A.G + kvh;
      sk = A.ks[at];
      sv = A.vs[at];
    }
  };
  auto store = [&](int stage) {
    const unsigned at = base + stage * L::STAGE;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int row = cr + i * (256 / CH);
      const unsigned kr = at + row * (D * 2), vr = kr + L::K;
      const int ksw = fl_kswz<D>(row), vsw = fl_vswz<D>(row);
      *fl_lds<c8_h8>(kr + ((2 * cc) ^ ksw) * 16) = c8_widen8<KIND>(kw[i].x, kw[i].y);
      *fl_lds<c8_h8>(kr + ((2 * cc + 1) ^ ksw) * 16) = c8_widen8<KIND>(kw[i].z, kw[i].w);
      *fl_lds<c8_h8>(vr + ((2 * cc) ^ vsw) * 16) = c8_widen8<KIND>(vw[i].x, vw[i].y);
      *fl_lds<c8_h8>(vr + ((2 * cc + 1) ^ vsw) * 16) = c8_widen8<KIND>(vw[i].z, vw[i].w);
    }
    if (tid < 4) {
      float* s = reinterpret_cast<float*>(lds + L::SCALES + stage * 64) + tid;
      const float vs = a8_least(sv);
      s[0] = there ? a8_least(sk) : 1.f;
      s[4] = there ? __builtin_amdgcn_logf(vs) : -INFINITY;
      s[8] = there ? 1.f / vs : 0.f;
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
  if (n > 0) {
    look(i0);
    fetch(i0);
    look(i0 + 1);
    store(0);
  }
  for (int i = 0; i < n; ++i) {
    const int stage = i & 1, kt = (i0 + i) * A8P_KEYS;
    if (i + 1 < n) {
      fetch(i0 + i + 1);
      look(i0 + i + 2);
    }
    __syncthreads();                                         // this stage is written; nobody reads the other one any more
    float16v s[2] = {zero, zero};
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*fl_lds<c8_h8>(kb[u] + stage * L::STAGE + 32 * t * D * 2), qf[u], s[t], 0, 0, 0);
    const float* sc = reinterpret_cast<const float*>(lds + L::SCALES + stage * 64);
    if (kt + A8P_KEYS > f.keys || (A.causal && kt + A8P_KEYS - 1 > f.past + (r0 + wave * 32) / Gq)) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int key = kt + 32 * t + (j & 3) + 8 * (j >> 2) + 4 * h;
          if (key >= f.keys || key > qpos) s[t][j] = -INFINITY;
        }
    }
    // t = x c + log2 vs with c above zero: the largest product of a group of 16 keys is its largest score
    float c[4], lv[4], mx = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float k = factor * sc[g];
      c[g] = k < 1.1754943508222875e-38f ? 1.1754943508222875e-38f : k;     // of no use to a masked -infinity if zero; NaN stays
      lv[g] = sc[4 + g];
      float x = s[g >> 1][8 * (g & 1)];
#pragma unroll
      for (int j = 1; j < 8; ++j) x = fmaxf(x, s[g >> 1][8 * (g & 1) + j]);
      mx = fmaxf(mx, fmaf(x, c[g], lv[g]));
    }
    const float m_new = fmaxf(m, fl_max32(mx));
    if (__any(m_new > m)) {
      const float alpha = __builtin_amdgcn_exp2f(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < NDT; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[d][j] *= alpha;
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      c8_h8 p;
      float sum = 0.f;
      const float off = lv[g] - m;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e = __builtin_amdgcn_exp2f(fmaf(s[g >> 1][8 * (g & 1) + j], c[g], off));
        sum += e;
        p[j] = (_Float16)e;
      }
      l = fmaf(sum, sc[8 + g], l);
#pragma unroll
      for (int d = 0; d < NDT; ++d) {
        const unsigned a = vb[d] + stage * L::STAGE + 16 * g * D * 2;
        const fl_v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(fl_lds<fl_v4s>(a));
        const fl_v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(fl_lds<fl_v4s>(a + 8 * D * 2));
        short8 a8;
#pragma unroll
        for (int j = 0; j < 4; ++j) { a8[j] = lo[j]; a8[4 + j] = hi[j]; }
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(c8_h8, a8), p, acc[d], 0, 0, 0);
      }
    }
    if (i + 1 < n) store(1 - stage);
  }
  l = fl_both32(l);                                          // a lane has summed up its half of the keys
  const size_t unit = ((size_t)b * A.G + kvh) * A.row_blocks + block;
  const bool whole = (((size_t)A.out | (size_t)A.ldo * 2) & 7) == 0;
  auto put = [&](int row, int c, const float4v& o, float ls) {
    const int t = (r0 + row) / Gq;
    a8_put(A.out + (size_t)(f.q0 + t) * A.ldo + (size_t)(kvh * Gq + r0 + row - t * Gq) * D + c, o, ls, whole);
  };
  const int row = wave * 32 + (lane & 31);
  const auto rs = a8_rsrc(A, nparts > 1 ? unit : 0, nparts > 1 ? part : 0, A8P_ROWS, D);
  if (row < rows) {
#pragma unroll
    for (int d = 0; d < NDT; ++d)
#pragma unroll
      for (int u = 0; u < 4; ++u) {                          // accumulators 4 u ..: columns 32 d + 8 u + 4 h ..
        const float4v o = {acc[d][4 * u], acc[d][4 * u + 1], acc[d][4 * u + 2], acc[d][4 * u + 3]};
        const int c = 32 * d + 8 * u + 4 * h;
        if (nparts == 1) put(row, c, o, l);
        else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(a8_u4, o), rs, (row * D + c) * 4, 0, 16);
      }
    if (nparts > 1 && h == 0) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(a8_u2, make_float2(m, l)), rs, (A8P_ROWS * D + 2 * row) * 4, 0, 16);
  }
  if (nparts == 1) return;
  if (!a8_last(A.tickets + unit * TICKET, nparts, reinterpret_cast<int*>(lds))) return;
  a8_join<D, A8P_ROWS, 256>(A, unit, nparts, rows, put);
}

// rows of a workgroup of the form that takes a call: 16 (tokens) or 128 (prompts)
extern "C" int loqa_attention8(const void* q, long ldq, const void* k, const void* v, const void* ks, const void* vs, const void* cu,
                               const void* ctx, const void* bt, void* out, long ldo, int T, int B, int H, int G, int D, int blk, int n_blocks,
                               int max_blocks, int max_q, float scale, int causal, int kind, int parts, void* ws, long ws_floats, void* tickets,
                               long n_tickets, hipStream_t st) {
  if (T <= 0 || B <= 0 || max_q <= 0) return 0;
  if ((D != 64 && D != 128) || (kind != C8_INT8 && kind != C8_E4M3) || blk < 16 || (blk & (blk - 1)) || G <= 0 || H <= 0 || H % G ||
      n_blocks <= 0 || max_blocks <= 0 || parts <= 0)
    return (int)hipErrorInvalidValue;
  const bool token = (long long)max_q * (H / G) <= A8_ROWS;
  const long long blocks = token ? 1 : ((long long)max_q * (H / G) + A8P_ROWS - 1) / A8P_ROWS, units = (long long)B * G * blocks;
  const int rows = token ? A8_ROWS : A8P_ROWS;
  if (token ? G > 65535 || B > 65535 || parts > 1 << 24 : units * parts > 1 << 30) return (int)hipErrorInvalidValue;
  if (blocks > 1 << 24 || (long long)parts * rows * (D + 2) * 4 >= 1LL << 31)
    return (int)hipErrorInvalidValue;
  if (parts > 1 && (!ws || !tickets || ws_floats < units * parts * rows * (D + 2) || n_tickets < units)) return (int)hipErrorInvalidValue;
  const Attn8Args a{(const bf16_t*)q, ldq, (const unsigned char*)k, (const unsigned char*)v, (const float*)ks, (const float*)vs, (const int*)cu,
                    (const int*)ctx, (const int*)bt, (bf16_t*)out, ldo, (float*)ws, (int*)tickets, T, B, H, G, __builtin_ctz(blk), n_blocks, max_blocks,
                    max_q, parts, causal, (int)blocks, units * parts <= 512, scale * 1.4426950408889634f};
  if (token) {
    const dim3 grid(parts, G, B);
#define GO(D_, K_) hipLaunchKernelGGL((attn8_token_kernel<D_, K_>), grid, dim3(A8_WAVES * 64), 0, st, a)
    if (D == 64) { if (kind == C8_INT8) GO(64, C8_INT8); else GO(64, C8_E4M3); }
    else { if (kind == C8_INT8) GO(128, C8_INT8); else GO(128, C8_E4M3); }
#undef GO
  } else {
    const dim3 grid((unsigned)(units * parts));
#define GO(D_, K_) hipLaunchKernelGGL((attn8_prompt_kernel<D_, K_>), grid, dim3(256), 0, st, a)
    if (D == 64) { if (kind == C8_INT8) GO(64, C8_INT8); else GO(64, C8_E4M3); }
    else { if (kind == C8_INT8) GO(128, C8_INT8); else GO(128, C8_E4M3); }
#undef GO
  }
  return (int)hipGetLastError();
}
