// Writing and reading the paged cache in 8 bits (cache8.h), and pages handed out on the GPU.
#include "cache8.h"

// ------------------------------------------------------------------ rotation and append
// Row i of sequence b stands at position ctx - n + i. Query heads are rotated to q_out; keys are rotated, keys and
// values rounded to codes of their page's scale
//
//   s = max(f(max |new rows of the page|), s before (if the page held rows), 2^-100),   f(a) = a / 127 or 2^ceil(log2(a / 448))
//
// in f32 from the bf16 rows to the one rounding (products and sums unfused and quotients rounded once, so that the codes are
// those of the CPU form bit for bit; torch on the GPU divides by 127 as a product with its reciprocal, and its int8 scales are an ulp off
// now and then). Where s grows, the page's older rows are rounded again to it.
// A wave has one page of one head, keys or values, and with it all that touches that scale: no atomics, and the
// same codes whatever else is in the batch. Bound by latency for token steps (metadata, page number, scale and rows
// one behind the other: eight replies x 32 + 2 x 8 heads of 128 4.7 us), by the bytes of qkv and q for prompts (2048 such rows, 46 MB, 11 us,
// 4.2 TB/s, the median of 12 calls under the profiler, 13 in another run; with each head's load behind the store of the one before, and keys and values last, 14.4; 16 bytes a load: no faster). Rows of a page are read once and kept where a wave has no more than AP_DEEP of them a lane (331 rows x 5, pages of 32 x 64
// columns 8.0 -> 6.4 us).
struct AppendArgs {
  const bf16_t* qkv;
  long long ld;
  const float* cs;
  int cs_rows;
  unsigned char *k, *v;
  float *ks, *vs;
  const int *cu, *ctx, *bt;
  bf16_t* q;
  long long ldq;
  int T, H, G, sh, n_blocks, max_blocks, max_q, kv_wgs;
};

#define AP_HEADS 4                                // query heads of a thread
#define AP_DEEP 4

template <int D> struct ApPair {                  // entries c, c + 1, c + 2, c + 3 of both halves of a row
  float4v a, b;
};

template <int D> __device__ __forceinline__ ApPair<D> ap_load(const bf16_t* row, int c) {
  const uint2 x = *reinterpret_cast<const uint2*>(row + c), y = *reinterpret_cast<const uint2*>(row + D / 2 + c);
  ApPair<D> p;
  p.a = float4v{__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xffff0000u)};
  p.b = float4v{__uint_as_float(y.x << 16), __uint_as_float(y.x & 0xffff0000u), __uint_as_float(y.y << 16), __uint_as_float(y.y & 0xffff0000u)};
  return p;
}

struct ApTurn { float4v c, s; };
template <int D> __device__ __forceinline__ ApTurn ap_turn(const AppendArgs& A, int pos, int c) {
  const float* t = A.cs + ((size_t)min(max(pos, 0), A.cs_rows - 1) * (D / 2) + c) * 2;
  const float4v x = *reinterpret_cast<const float4v*>(t), y = *reinterpret_cast<const float4v*>(t + 4);
  return ApTurn{float4v{x[0], x[2], y[0], y[2]}, float4v{x[1], x[3], y[1], y[3]}};
}

template <int D> __device__ __forceinline__ void ap_rotate(ApPair<D>& p, const ApTurn& t) {
#pragma clang fp contract(off)
  const float4v a = p.a, b = p.b;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p.a[i] = a[i] * t.c[i] - b[i] * t.s[i];
    p.b[i] = b[i] * t.c[i] + a[i] * t.s[i];
  }
}

template <int D, int KIND>
__global__ __launch_bounds__(256) void rope_append8_kernel(AppendArgs A) {
  constexpr int LPR = D / 8, RPW = 64 / LPR;      // lanes of a row, rows of a wave at once
  const int b = blockIdx.y;
  const int q0 = min(max(A.cu[b], 0), A.T), fed = min(max(A.cu[b + 1], q0), A.T) - q0;
  const int n = min(fed, A.max_q), start = A.ctx[b] - fed, end = start + n;
  if ((int)blockIdx.x >= A.kv_wgs) {              // keys and values, whose chain of loads is the longer, come first
    const int chunks = (A.H + AP_HEADS - 1) / AP_HEADS, id = (blockIdx.x - A.kv_wgs) * 256 + threadIdx.x;
    const int c = id % LPR * 4, unit = id / LPR, i = unit / chunks, h0 = unit % chunks * AP_HEADS;
    if (i >= n) return;
    ApTurn t;
    if (A.cs) t = ap_turn<D>(A, start + i, c);
    const bf16_t* row = A.qkv + (size_t)(q0 + i) * A.ld;
    bf16_t* out = A.q + (size_t)(q0 + i) * A.ldq;
    ApPair<D> pairs[AP_HEADS];                    // all asked for ahead of the first store, which q_out may lie in their place
#pragma unroll
    for (int u = 0; u < AP_HEADS; ++u) pairs[u] = ap_load<D>(row + min(h0 + u, A.H - 1) * D, c);
#pragma unroll
    for (int u = 0; u < AP_HEADS; ++u) {
      if (h0 + u >= A.H) break;
      ApPair<D>& p = pairs[u];
      if (A.cs) ap_rotate<D>(p, t);
      *reinterpret_cast<uint2*>(out + (h0 + u) * D + c) = make_uint2(pack_bf16x2(p.a[0], p.a[1]), pack_bf16x2(p.a[2], p.a[3]));
      *reinterpret_cast<uint2*>(out + (h0 + u) * D + D / 2 + c) = make_uint2(pack_bf16x2(p.b[0], p.b[1]), pack_bf16x2(p.b[2], p.b[3]));
    }
    return;
  }
  const int lane = threadIdx.x & 63;
  const int w = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int values = w & 1, g = (w >> 1) % A.G, pj = (max(start, 0) >> A.sh) + (w >> 1) / A.G;
  const int lo = max(start, pj << A.sh);
  if (n <= 0 || pj >= A.max_blocks || lo >= end) return;
  const int hi = min(end, (pj + 1) << A.sh), off = lo - (pj << A.sh), rows = hi - lo;
  const int page = A.bt[(size_t)b * A.max_blocks + pj];
  if ((unsigned)page >= (unsigned)A.n_blocks) return;
  const size_t at = (size_t)page * A.G + g;
  float* scale = (values ? A.vs : A.ks) + at;
  unsigned char* codes = (values ? A.v : A.k) + ((at << A.sh) * D);
  const bool turn = A.cs && !values;
  const int c = lane % LPR * 4, r0 = lane / LPR;
  const bf16_t* src = A.qkv + (size_t)(q0 + lo - start) * A.ld + (size_t)(A.H + (values ? A.G : 0) + g) * D;
  const float before = off > 0 ? *scale : 0.f;
  const unsigned had = off > 0 ? __float_as_uint(c8_least(before)) & 0x7fffffffu : 0u;
  // AP_DEEP rows of a lane under way together; a page of no more than that is read once
  constexpr int DEEP = AP_DEEP * RPW;
  ApPair<D> p[AP_DEEP];
  auto take = [&](int at) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < AP_DEEP; ++i) p[i] = ap_load<D>(src + (size_t)min(at + i * RPW + r0, rows - 1) * A.ld, c);
    if (turn) {
      ApTurn t[AP_DEEP];
#pragma unroll
      for (int i = 0; i < AP_DEEP; ++i) t[i] = ap_turn<D>(A, lo + min(at + i * RPW + r0, rows - 1), c);
#pragma unroll
      for (int i = 0; i < AP_DEEP; ++i) ap_rotate<D>(p[i], t[i]);
    }
  };
  // magnitudes as whole numbers: infinities and NaN are the largest (rows behind the last one are the last once more)
  unsigned top = 0;
  for (int at = 0; at < rows; at += DEEP) {
    take(at);
#pragma unroll
    for (int u = 0; u < AP_DEEP; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max(top, max(__float_as_uint(p[u].a[i]) & 0x7fffffffu, __float_as_uint(p[u].b[i]) & 0x7fffffffu));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
  const unsigned now = max(max(c8_scale<KIND>(top), had), __float_as_uint(C8_LEAST));
  const float s = __uint_as_float(now), s_had = __uint_as_float(had);
  if (off > 0 && now != had)
    for (int r = r0; r < off; r += RPW) {
      uint2* p = reinterpret_cast<uint2*>(codes + r * D + lane % LPR * 8);
      const uint2 x = *p;
      float4v f[2] = {c8_floats<KIND>(x.x), c8_floats<KIND>(x.y)};
#pragma unroll
      for (int i = 0; i < 4; ++i) { f[0][i] *= s_had; f[1][i] *= s_had; }
      *p = make_uint2(c8_codes<KIND>(f[0], s), c8_codes<KIND>(f[1], s));
    }
  for (int at = 0; at < rows; at += DEEP) {
    if (rows > DEEP) take(at);
#pragma unroll
    for (int i = 0; i < AP_DEEP; ++i) {
      const int r = at + i * RPW + r0;
      if (r >= rows) continue;
      *reinterpret_cast<unsigned*>(codes + (off + r) * D + c) = c8_codes<KIND>(p[i].a, s);
      *reinterpret_cast<unsigned*>(codes + (off + r) * D + D / 2 + c) = c8_codes<KIND>(p[i].b, s);
    }
  }
  if (lane == 0 && (off == 0 || now != __float_as_uint(before))) *scale = s;
}

extern "C" int loqa_rope_append8(const void* qkv, long ld, const void* cs, int cs_rows, void* k, void* v, void* ks, void* vs, const void* cu,
                                 const void* ctx, const void* bt, void* q, long ldq, int T, int B, int H, int G, int D, int blk, int n_blocks,
                                 int max_blocks, int max_q, int kind, hipStream_t st) {
  if (T <= 0 || B <= 0 || max_q <= 0) return 0;
  if ((D != 64 && D != 128) || (kind != C8_INT8 && kind != C8_E4M3) || blk < 16 || (blk & (blk - 1)) || B > 65535 || H <= 0 || G <= 0 ||
      n_blocks <= 0 || max_blocks <= 0 || (cs && cs_rows <= 0) || ld % 4 || ldq % 4)
    return (int)hipErrorInvalidValue;
  AppendArgs a{(const bf16_t*)qkv, ld, (const float*)cs, cs_rows, (unsigned char*)k, (unsigned char*)v, (float*)ks, (float*)vs, (const int*)cu,
               (const int*)ctx, (const int*)bt, (bf16_t*)q, ldq, T, H, G, __builtin_ctz(blk), n_blocks, max_blocks, max_q, 0};
  const long long units = (long long)max_q * ((H + AP_HEADS - 1) / AP_HEADS) * (D / 8);
  const long long pages = ((long long)max_q + blk - 2) / blk + 1, waves = pages * G * 2;   // a feed touches that many pages at most
  const long long wgs = (units + 255) / 256 + (waves + 3) / 4;
  if (units > 1LL << 30 || wgs > 1LL << 24) return (int)hipErrorInvalidValue;
  a.kv_wgs = (int)((waves + 3) / 4);
  const dim3 grid((unsigned)wgs, B);
#define GO(D_, K_) hipLaunchKernelGGL((rope_append8_kernel<D_, K_>), grid, dim3(256), 0, st, a)
  if (D == 64) { if (kind == C8_INT8) GO(64, C8_INT8); else GO(64, C8_E4M3); }
  else { if (kind == C8_INT8) GO(128, C8_INT8); else GO(128, C8_E4M3); }
#undef GO
  return (int)hipGetLastError();
}

// ------------------------------------------------------------------ rows back
// Row cu[b] + i of the results is position first[b] + i of sequence b, in bf16 (code * scale, rounded once);
// zeros from a page that does not exist and in rows of no sequence. A thread has eight entries of keys and of values;
// bound by what it writes (2048 rows x 8 heads of 128, 12.6 MB, 4.7 us).
struct Read8Args {
  const unsigned char *k, *v;
  const float *ks, *vs;
  const int *cu, *first, *bt;
  bf16_t *ko, *vo;
  int total, B, G, sh, n_blocks, max_blocks;
};

template <int D, int KIND>
__global__ __launch_bounds__(256) void read8_kernel(Read8Args A) {
  constexpr int C = D / 8;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long t64 = id / (C * A.G);
  if (t64 >= A.total) return;
  const int t = (int)t64, g = (int)(id / C % A.G), c = (int)(id % C);
  int lo = 0, hi = A.B;                           // the last b with cu[b] <= t
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (A.cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  const bool in = t >= A.cu[lo] && t < A.cu[lo + 1];
  const int pos = A.first[lo] + t - A.cu[lo];
  const int pj = pos >> A.sh, page = !in || pos < 0 || pj >= A.max_blocks ? -1 : A.bt[(size_t)lo * A.max_blocks + pj];
  uint4 ko = make_uint4(0, 0, 0, 0), vo = ko;
  if ((unsigned)page < (unsigned)A.n_blocks) {
    const size_t at = (size_t)page * A.G + g, off = ((at << A.sh) + (pos & ((1 << A.sh) - 1))) * D + c * 8;
    const uint2 x = *reinterpret_cast<const uint2*>(A.k + off), y = *reinterpret_cast<const uint2*>(A.v + off);
    const float sk = c8_least(A.ks[at]), sv = c8_least(A.vs[at]);
    const float4v a = c8_floats<KIND>(x.x), b = c8_floats<KIND>(x.y), e = c8_floats<KIND>(y.x), f = c8_floats<KIND>(y.y);
    ko = make_uint4(pack_bf16x2(a[0] * sk, a[1] * sk), pack_bf16x2(a[2] * sk, a[3] * sk), pack_bf16x2(b[0] * sk, b[1] * sk), pack_bf16x2(b[2] * sk, b[3] * sk));
    vo = make_uint4(pack_bf16x2(e[0] * sv, e[1] * sv), pack_bf16x2(e[2] * sv, e[3] * sv), pack_bf16x2(f[0] * sv, f[1] * sv), pack_bf16x2(f[2] * sv, f[3] * sv));
  }
  const size_t to = ((size_t)t * A.G + g) * D + c * 8;
  *reinterpret_cast<uint4*>(A.ko + to) = ko;
  *reinterpret_cast<uint4*>(A.vo + to) = vo;
}

extern "C" int loqa_read8(const void* k, const void* v, const void* ks, const void* vs, const void* cu, const void* first, const void* bt, void* ko,
                          void* vo, int total, int B, int G, int D, int blk, int n_blocks, int max_blocks, int kind, hipStream_t st) {
  if (total <= 0 || B <= 0) return 0;
  if ((D != 64 && D != 128) || (kind != C8_INT8 && kind != C8_E4M3) || blk < 16 || (blk & (blk - 1)) || G <= 0 || n_blocks <= 0 || max_blocks <= 0)
    return (int)hipErrorInvalidValue;
  const Read8Args a{(const unsigned char*)k, (const unsigned char*)v, (const float*)ks, (const float*)vs, (const int*)cu, (const int*)first,
                    (const int*)bt, (bf16_t*)ko, (bf16_t*)vo, total, B, G, __builtin_ctz(blk), n_blocks, max_blocks};
  const long long wgs = ((long long)total * G * (D / 8) + 255) / 256;
  if (wgs > 1LL << 30) return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)wgs);
#define GO(D_, K_) hipLaunchKernelGGL((read8_kernel<D_, K_>), grid, dim3(256), 0, st, a)
  if (D == 64) { if (kind == C8_INT8) GO(64, C8_INT8); else GO(64, C8_E4M3); }
  else { if (kind == C8_INT8) GO(128, C8_INT8); else GO(128, C8_E4M3); }
#undef GO
  return (int)hipGetLastError();
}

// ------------------------------------------------------------------ pages and slots of a step
// c tokens of sequence i are cached in its first ceil(c / P) table entries and n more come (n = -1: it has ended):
//
//   want = ceil((c + n) / P) - ceil(c / P) entries from the ring of free pages, in the order of the sequences,
//   back = ceil(c / P) entries of an ended one to the ring's end,
//
// cu, first and given the sums of n, want and back ahead of i. Every workgroup sums up all sequences in LDS (a few
// KB, from L2) and takes its part of the tokens, of the entries handed out and of those given back, each found by
// bisection of the sums; a token's page follows from the ring itself, so nothing waits for the table. What a caller may
// update in place (lengths, the ring's head and count) is written by the last workgroup to have read it (without a ticket there
// is one workgroup).
// All or nothing: with a status nothing changes. Bound by its launch and the chain metadata, sums, ring, slots: 4.1 us for eight
// sequences of a token each. 500 of them take 5.7, one pass of the sums too, but nine steps of each bisection and 500 entries of every
// output; as many with 6000 tokens 6.5, with 32000 7.2: a token's bisection, its 64-bit remainder and the page that it then asks for, and up to
// 64 workgroups that meet at one ticket. (Eight sequences with 24000 tokens 5.4.)
struct PageArgs {
  const int *n, *ctx;
  int* table;
  int* free_;
  const int* ring;
  int *cu, *pos, *slots;
  long long* last;
  int *ctx_out, *ring_out, *status;
  int* ticket;
  int B, width, sh, pool, most;
};

#define PS_THREADS 512
#define PS_SEQS 4096

struct PsSum { long long fed, want, back; };
__device__ __forceinline__ PsSum ps_up(const PsSum& s, int o) {
  return PsSum{__shfl_up(s.fed, o, 64), __shfl_up(s.want, o, 64), __shfl_up(s.back, o, 64)};
}

__global__ __launch_bounds__(PS_THREADS) void page_step_kernel(PageArgs A) {
  // sums ahead of each sequence; ctx, cu and held of it for the tokens
  __shared__ int cu[PS_SEQS + 1], first[PS_SEQS + 1], given[PS_SEQS + 1], len[PS_SEQS];
  __shared__ PsSum part[PS_THREADS / 64];
  __shared__ int bad_s, last_s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, B = A.B, P = 1 << A.sh;
  if (tid == 0) bad_s = 0;
  __syncthreads();
  const int head = A.ring[0], count = A.ring[1];
  PsSum run{0, 0, 0};
  int bad = head < 0 || head >= A.pool || count < 0 || count > A.pool ? 8 : 0;
  for (int i0 = 0; i0 < B; i0 += PS_THREADS) {
    const int i = i0 + tid;
    PsSum s{0, 0, 0};
    int c = 0;
    if (i < B) {
      const int n = A.n[i];
      c = A.ctx[i];
      const long long fed = n > 0 ? n : 0, held = ((long long)c + P - 1) >> A.sh;
      if (n < -1 || c < 0) bad |= 8;
      if (c + fed > (long long)A.width * P) bad |= 4;
      s = PsSum{fed, ((c + fed + P - 1) >> A.sh) - held, n == -1 ? held : 0};
    }
    PsSum x = s;                                  // inclusive sums of the wave, then ahead of it
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const PsSum y = ps_up(x, o);
      if (lane >= o) { x.fed += y.fed; x.want += y.want; x.back += y.back; }
    }
    if (lane == 63) part[wave] = x;
    __syncthreads();
    PsSum all = run;
    for (int w = 0; w < PS_THREADS / 64; ++w) {
      if (w == wave) { x.fed += all.fed; x.want += all.want; x.back += all.back; }
      all.fed += part[w].fed; all.want += part[w].want; all.back += part[w].back;
    }
    if (i < B) {
      cu[i] = (int)(x.fed - s.fed);
      first[i] = (int)(x.want - s.want);
      given[i] = (int)(x.back - s.back);
      len[i] = c;
    }
    run = all;
    __syncthreads();
  }
  if (run.want > count) bad |= 1;
  if (run.fed > A.most) bad |= 2;
  if (run.back + count > A.pool) bad |= 8;        // more pages than there are
  if (bad) atomicOr(&bad_s, bad);
  if (tid == 0) { cu[B] = (int)run.fed; first[B] = (int)run.want; given[B] = (int)run.back; }
  __syncthreads();
  bad = bad_s;
  // every workgroup is through with lengths and ring: the last one may write them
  if (tid == 0 && gridDim.x == 1) last_s = 1;
  else if (tid == 0) {
    const int t = __hip_atomic_fetch_add(A.ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last_s = t == (int)gridDim.x - 1;
    if (last_s) __hip_atomic_store(A.ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (last_s) {
    for (int i = tid; i <= B; i += PS_THREADS) {
      A.cu[i] = bad ? 0 : cu[i];
      if (i < B) {
        const int fed = cu[i + 1] - cu[i], gone = given[i + 1] - given[i];
        // an ended sequence without pages has no length to lose
        A.ctx_out[i] = bad ? len[i] : gone ? 0 : len[i] + fed;
        A.last[i] = bad || fed == 0 ? 0 : cu[i + 1] - 1;
      }
    }
    if (tid == 0) {
      A.ring_out[0] = bad ? head : (int)(((long long)head + run.want) % A.pool);
      A.ring_out[1] = bad ? count : (int)(count - run.want + run.back);
      A.status[0] = bad;
    }
  }
  auto find = [&](const int* sums, int t) {       // the last i with sums[i] <= t: a sequence that has t
    int lo = 0, hi = B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (sums[mid] <= t) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  const int id = blockIdx.x * PS_THREADS + tid, step = gridDim.x * PS_THREADS;
  const int fed = bad ? 0 : (int)run.fed;
  for (int t = id; t < A.most; t += step) {
    int p = 0, slot = -1;
    if (t < fed) {
      const int i = find(cu, t);
      p = len[i] + t - cu[i];
      const int j = p >> A.sh, held = (len[i] + P - 1) >> A.sh;
      const int page = j < held ? A.table[(size_t)i * A.width + j] : A.free_[((long long)head + first[i] + j - held) % A.pool];
      slot = (int)((unsigned)page * (unsigned)P + (p & (P - 1)));
    }
    A.pos[t] = p;
    A.slots[t] = slot;
  }
  if (bad) return;
  for (int e = id; e < (int)run.want; e += step) {
    const int i = find(first, e);
    A.table[(size_t)i * A.width + ((len[i] + P - 1) >> A.sh) + e - first[i]] = A.free_[((long long)head + e) % A.pool];
  }
  for (int e = id; e < (int)run.back; e += step) {
    const int i = find(given, e);
    A.free_[((long long)head + count + e) % A.pool] = A.table[(size_t)i * A.width + e - given[i]];
  }
}

extern "C" int loqa_page_step(const void* n, const void* ctx, void* table, void* free_, const void* ring, void* cu, void* pos, void* slots,
                              void* last, void* ctx_out, void* ring_out, void* status, void* ticket, int B, int width, int blk, int pool,
                              int most, hipStream_t st) {
  if (B <= 0 || B > PS_SEQS || width <= 0 || blk <= 0 || (blk & (blk - 1)) || pool <= 0 || most < 0 || most > 1 << 30) return (int)hipErrorInvalidValue;
  const PageArgs a{(const int*)n, (const int*)ctx, (int*)table, (int*)free_, (const int*)ring, (int*)cu, (int*)pos, (int*)slots, (long long*)last,
                   (int*)ctx_out, (int*)ring_out, (int*)status, (int*)ticket, B, width, __builtin_ctz(blk), pool, most};
  const int wgs = ticket ? max(1, min(64, (most + PS_THREADS - 1) / PS_THREADS)) : 1;
  hipLaunchKernelGGL(page_step_kernel, dim3(wgs), dim3(PS_THREADS), 0, st, a);
  return (int)hipGetLastError();
}
