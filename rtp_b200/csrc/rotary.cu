// Rotary positions of queries and keys: of every head the first `rot` elements form pairs, and pair i of a token at position p
// turns by the angle p * f_i:
//     (a, b) -> m * (a cos - b sin, a sin + b cos)
// with pairs (x[i], x[i + rot / 2]) in the half layout and (x[2 i], x[2 i + 1]) in the interleaved one; the elements behind `rot`
// are copied.  Backward is the transposed map: the same kernel with the sine negated.
//
// The angle is made here from the position and the frequency in 64 bits (at position 10^6 an fp32 product is off by 0.06 rad), taken
// modulo a whole turn and only then rounded, so positions know no bound and no table is read.  One block takes a few tokens: its
// threads make the cosines and sines of those tokens into shared memory once, for all heads of q and k.
//
// Bound by memory: every element is read and written once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "common.cuh"
#include "kernels.h"
#include "launch.h"

namespace {
using namespace rtp;

thread_local std::string g_err;
int fail(const std::string& s) { g_err = s; return -1; }

constexpr int kThreads = 256;
constexpr int kMaxTile = 64;              // tokens of a block
constexpr int kMaxTrig = 2048;            // their (cosine, sine) pairs: 16 KB

struct Side {                             // q or k: [B, S, heads, hd] views in and out (out may be in)
  const void* in;
  void* out;
  long long sb, ss, sh, osb, oss, osh;
  int heads;
};
struct Params {
  Side q, k;
  const void* positions;
  long long pb, ps;
  int pos64;
  const double* freqs;
  float magnitude, sign;
  long long tokens;
  int S, hd, rot, tile, per_head, rows_per_pass;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec { T e[V]; };

// V: elements of one access.  HALF: an item is V pairs (two accesses) or V copied elements; otherwise max(V, 2) consecutive ones.
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ Params p) {
  __shared__ __align__(16) float s_cos[kMaxTrig], s_sin[kMaxTrig];
  __shared__ long long s_at[2][2][kMaxTile];                // [q, k][in, out]: where a token begins
  pdl_prologue();
  const long long t0 = blockIdx.x * (long long)p.tile;
  const int n = (int)min((long long)p.tile, p.tokens - t0), half = p.rot >> 1, tid = threadIdx.x;
  for (int i = tid; i < n * half; i += kThreads) {
    const int t = i / half, c = i - t * half;
    const long long tok = t0 + t, b = tok / p.S, s = tok - b * p.S, at = b * p.pb + s * p.ps;
    const double pos = p.pos64 ? (double)reinterpret_cast<const long long*>(p.positions)[at]
                               : (double)reinterpret_cast<const int*>(p.positions)[at];
    const double turns = pos * p.freqs[c] * 0.15915494309189533577;
    float sn, cs;
    sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
    s_cos[i] = cs * p.magnitude;
    s_sin[i] = sn * p.magnitude * p.sign;
  }
  for (int t = tid; t < n; t += kThreads) {
    const long long b = (t0 + t) / p.S, s = t0 + t - b * p.S;
    s_at[0][0][t] = b * p.q.sb + s * p.q.ss;
    s_at[0][1][t] = b * p.q.osb + s * p.q.oss;
    s_at[1][0][t] = b * p.k.sb + s * p.k.ss;
    s_at[1][1][t] = b * p.k.osb + s * p.k.oss;
  }
  __syncthreads();
  const int row0 = tid / p.per_head, j = tid - row0 * p.per_head;
  if (row0 >= p.rows_per_pass) return;
  const int heads = p.q.heads + p.k.heads;
  using W = Vec<T, V>;
  int t = row0 / heads, h = row0 - t * heads;
  while (t < n) {
    const bool is_q = h < p.q.heads;
    const Side& sd = is_q ? p.q : p.k;
    const int hh = is_q ? h : h - p.q.heads;
    const T* in = reinterpret_cast<const T*>(sd.in) + s_at[!is_q][0][t] + hh * sd.sh;
    T* out = reinterpret_cast<T*>(sd.out) + s_at[!is_q][1][t] + hh * sd.osh;
    const float *cs = s_cos + t * half, *sn = s_sin + t * half;
    if constexpr (HALF) {
      const int c = j * V;
      if (c < half) {
        W a = *reinterpret_cast<const W*>(in + c), b = *reinterpret_cast<const W*>(in + half + c);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float x = to_f(a.e[e]), y = to_f(b.e[e]), co = cs[c + e], si = sn[c + e];
          a.e[e] = from_f<T>(x * co - y * si);
          b.e[e] = from_f<T>(x * si + y * co);
        }
        *reinterpret_cast<W*>(out + c) = a;
        *reinterpret_cast<W*>(out + half + c) = b;
      } else {
        *reinterpret_cast<W*>(out + half + c) = *reinterpret_cast<const W*>(in + half + c);
      }
    } else if constexpr (V == 1) {
      const int c = j * 2;
      T a = in[c], b = in[c + 1];
      if (c < p.rot) {
        const float x = to_f(a), y = to_f(b), co = cs[j], si = sn[j];
        a = from_f<T>(x * co - y * si);
        b = from_f<T>(x * si + y * co);
      }
      out[c] = a;
      out[c + 1] = b;
    } else {
      const int c = j * V;
      W a = *reinterpret_cast<const W*>(in + c);
      if (c < p.rot) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
          const float x = to_f(a.e[e]), y = to_f(a.e[e + 1]), co = cs[(c + e) >> 1], si = sn[(c + e) >> 1];
          a.e[e] = from_f<T>(x * co - y * si);
          a.e[e + 1] = from_f<T>(x * si + y * co);
        }
      }
      *reinterpret_cast<W*>(out + c) = a;
    }
    h += p.rows_per_pass;
    while (h >= heads) { h -= heads; ++t; }
  }
}

// q or k as the kernel sees it: strides of a single batch entry, position or head do not matter.
Side side(const RtpRotary& a, const void* in, void* out, const long long* st, const long long* ost, int heads) {
  const bool b = a.B > 1, s = a.S > 1, h = heads > 1;
  return Side{in, out, b ? st[0] : 0, s ? st[1] : 0, h ? st[2] : 0, b ? ost[0] : 0, s ? ost[1] : 0, h ? ost[2] : 0, heads};
}
// The widest access (bytes) that pairs, tail, strides and addresses allow.
int access_bytes(const RtpRotary& a, const Side& q, const Side& k, int size) {
  for (int bytes = 16; bytes > size; bytes >>= 1) {
    const int v = bytes / size;
    auto fits = [&](const Side& x) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(x.in) | reinterpret_cast<uintptr_t>(x.out);
      return !x.heads || (at % bytes == 0 && (x.sb | x.ss | x.sh | x.osb | x.oss | x.osh) % v == 0);
    };
    if (a.hd % v == 0 && (a.half_layout ? a.rot / 2 : a.rot) % v == 0 && fits(q) && fits(k)) return bytes;
  }
  return size;
}

template <typename T, int V>
cudaError_t launch(const Params& P, bool half, unsigned blocks, cudaStream_t s) {
  return launch_k(half ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>, dim3(blocks), dim3(kThreads), 0, s, P);
}

}  // namespace

extern "C" {

const char* rtp_rotary_last_error(void) { return g_err.c_str(); }

int rtp_rotary(const RtpRotary* a, void* stream) {
  if (a->B < 0 || a->S < 0 || a->q_heads < 0 || a->k_heads < 0) return fail("rotary: negative size");
  if (a->hd < 2 || a->hd % 2 || a->hd > 256) return fail("rotary: head_dim must be even and at most 256");
  if (a->rot < 2 || a->rot % 2 || a->rot > a->hd) return fail("rotary: the rotated part must be even and lie inside the head");
  if (a->dtype < 0 || a->dtype > 2) return fail("rotary: unknown element type");
  const long long tokens = (long long)a->B * a->S;
  const int heads = a->q_heads + a->k_heads;
  if (!tokens || !heads) return 0;
  Params P = {};
  P.q = side(*a, a->q, a->qo, a->q_st, a->qo_st, a->q_heads);
  P.k = side(*a, a->k, a->ko, a->k_st, a->ko_st, a->k_heads);
  const int size = a->dtype == 2 ? 4 : 2, bytes = access_bytes(*a, P.q, P.k, size), v = bytes / size;
  P.positions = a->positions; P.pb = a->pos_sb; P.ps = a->pos_ss; P.pos64 = a->pos64;
  P.freqs = a->freqs; P.magnitude = a->magnitude; P.sign = a->backward ? -1.f : 1.f;
  P.tokens = tokens; P.S = a->S; P.hd = a->hd; P.rot = a->rot;
  P.per_head = a->half_layout ? a->rot / 2 / v + (a->hd - a->rot) / v : a->hd / std::max(v, 2);
  P.rows_per_pass = kThreads / P.per_head;
  // tokens of a block: a few items a thread, as long as every SM has blocks enough
  const long long items = (long long)heads * P.per_head;
  long long tile = std::max(1ll, 4 * kThreads / items);
  tile = std::min({tile, std::max(1ll, tokens / (148 * 8)), (long long)kMaxTile, (long long)(2 * kMaxTrig / a->rot)});
  P.tile = (int)tile;
  const long long blocks = (tokens + tile - 1) / tile;
  if (blocks > 0x7fffffffll) return fail("rotary: too many tokens");
  const bool half = a->half_layout != 0;
  cudaStream_t s = (cudaStream_t)stream;
  const unsigned g = (unsigned)blocks;
  cudaError_t e;
  if (a->dtype == 2) e = v == 4 ? launch<float, 4>(P, half, g, s) : v == 2 ? launch<float, 2>(P, half, g, s) : launch<float, 1>(P, half, g, s);
  else if (a->dtype == 1)
    e = v == 8 ? launch<__half, 8>(P, half, g, s) : v == 4 ? launch<__half, 4>(P, half, g, s)
      : v == 2 ? launch<__half, 2>(P, half, g, s) : launch<__half, 1>(P, half, g, s);
  else
    e = v == 8 ? launch<__nv_bfloat16, 8>(P, half, g, s) : v == 4 ? launch<__nv_bfloat16, 4>(P, half, g, s)
      : v == 2 ? launch<__nv_bfloat16, 2>(P, half, g, s) : launch<__nv_bfloat16, 1>(P, half, g, s);
  return e == cudaSuccess ? 0 : fail(std::string("rotary: ") + cudaGetErrorString(e));
}

}  // extern "C"
