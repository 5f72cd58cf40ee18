// Attention backward for gfx950: dQ, dK and dV of O = softmax(scale Q K^T) V, recomputing P from the
// forward's log-sum-exp.
//
//   P = exp(scale Q K^T - lse)            (0 above the diagonal when causal)
//   delta_i = sum_d dO_id O_id - dlse_i,  dP = dO V^T,  dS = P (dP - delta)
//   dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K      (dK, dV summed over a group's query heads)
//
// Three products share each operand tile's two readings (rows for the products over D, transposed for the
// products over rows), and none of P, dP, dS leaves the registers:
//  * dK/dV blocks own 32 keys per wave. S = Q K^T with Q as the A operand gives each lane one key
//    (lane & 15) and four consecutive query rows per 16x16 tile, which is the B operand of
//    dV^T = dO^T P and dK^T = Q^T dS as it stands (two 16-row tiles make one k = 32 operand; the transposing
//    LDS read ds_read_b64_tr_b16 takes the matching rows). K, V and both sums stay in registers; Q and dO
//    tiles of 32 rows pass through LDS.
//  * dQ blocks own 32 query rows per wave: S^T = K Q^T, then dQ^T = K^T dS^T, with Q, dO and dQ in registers
//    and K, V tiles of 32 keys passing through LDS.
// Recomputing S and dP for dQ costs two more products than the five of a single pass, and buys sums in a
// fixed order (no atomics), no fp32 dQ in memory and no third pass to convert it.
//
// What bounds it. Per 32 x 32 step a wave makes 64 (dK/dV) or 48 (dQ) MFMAs of 16 cycles at D = 128 against 93 or 100
// vector instructions, 16 of them exponentials, and every Q, dO, K or V fragment read from LDS feeds two MFMAs:
// 128 bytes of LDS a cycle and CU at the full matrix rate. fp16 B4 H32 D128 N8192 takes 13.4 to 13.9 ms by card: 790 to
// 820 TFLOP/s of the five products, 1105 to 1150 of the seven executed, where an 8192-cube product reaches 1345 once the
// clock is up. The matrix rate is not the bound: the matrix pipes are busy 59% of cycles, waves wait 29% of theirs for a
// counter or barrier and 34% to issue. bf16 D256 N2048: 918 executed, pipes busy 39% (one wave per SIMD: nothing covers its
// softmax and its own LDS reads). Short sequences pay for each workgroup's own operands and gradients (a quarter of the
// time at N2048 causal, 580 to 605 us), few heads for the partial sums and for parts of unequal length: causal blocks
// have from all tiles to one block's, and all are cut into as many parts as the longest (bf16 B1 12/2 heads N4096, 241 us).
// Tried and slower: 64 rows per wave at D = 128 (half the LDS reads, but one wave per SIMD: 17.0 against 13.5 ms),
// three and four ring stages, reads scheduled ahead by hand, heavy and light causal blocks in pairs.
//
// fp16 range. P and dS enter the second products as 16-bit values. With fp16, P of long rows and dS of small
// gradients would fall under 2^-14 and lose bits, so P is scaled by 2^15 (in the exponent's offset, free)
// and dS by a power of two from a bound on |dP - delta| (row norms of dO and V, |delta|) that puts it under
// 2^15; the sums are scaled back in fp32. In dQ blocks a lane's products are all of one row, and the power is the
// row's own; in dK/dV blocks it is that of the largest row which the block's keys meet, and a row 2^k smaller keeps its
// bits down to weights of 2^(k - 29). bf16 has fp32's range and takes neither.
#include <type_traits>

#include "fa_common.h"
#include "fa_kernels.h"
#include "../../include/fa_gfx950.h"

namespace fa {

template <typename Tag>
struct BwdTraits;
template <>
struct BwdTraits<f16_t> {
  static constexpr bool kScaled = true;
  static constexpr float kPBias = 15.f;           // log2 of P's scale
  static constexpr float kPUnscale = 1.f / 32768.f;
};
template <>
struct BwdTraits<bf16_t> {
  static constexpr bool kScaled = false;
  static constexpr float kPBias = 0.f;
  static constexpr float kPUnscale = 1.f;
};

// Per-row terms in the workspace, in groups of 32 rows (one LDS-DMA of 4 bytes per lane):
// nd[bh][row / 32][0][32] = P's scale in log2 units - lse * log2(e) (-inf for a row that has no P: padding, no keys),
// nd[bh][row / 32][1][32] = -delta.
__device__ inline int64_t nd_index(const BwdParams& p, int64_t bh, int row) {
  return (bh * p.row_groups + (row >> 5)) * 64 + (row & 31);
}

constexpr int kPrepRows = 64;  // rows per block of the row-term kernel

// Row terms, and for fp16 the block maxima behind dS's scale: bound[0][bh][block] = max |dO row|^2,
// bound[1][bh][block] = max |delta|, vbound[b * Hkv + h][block] = max |V row|^2. Rows that are not finite
// are left out (their gradients are not finite whatever the scale is). Bound by memory: dO and O (fp16: V too) are
// read once, 201 MB in 31 us at B4 H32 N2048 D128.
template <typename Tag, int D>
__global__ __launch_bounds__(256) void fa_bwd_prep_kernel(BwdParams p) {
  constexpr int LPR = D / 8;          // lanes per row (16-byte loads)
  constexpr int RPP = 256 / LPR;      // rows per pass
  const int t = threadIdx.x, part = t % LPR, r0 = t / LPR;
  __shared__ float red[8];
  const uint32_t qblocks = p.prep_blocks, nq = (uint32_t)p.B * p.H * qblocks, id = blockIdx.x;
  constexpr int NP = 2;  // passes whose loads are issued together (four take a third longer: fewer waves fit)
  float top = 0.f, topd = 0.f;
  if (id < nq) {
    const uint32_t bh = id / qblocks;
    const int blk = (int)(id % qblocks), b = (int)(bh / (uint32_t)p.H), h = (int)(bh % (uint32_t)p.H);
    const uint16_t* ob = p.o + b * p.so[0] + h * p.so[1] + part * 8;
    const uint16_t* gb = p.dout + b * p.sdo[0] + h * p.sdo[1] + part * 8;
#pragma unroll 1
    for (int at = r0; at < kPrepRows; at += NP * RPP) {
      u32x4 x[NP], y[NP];
      float lse[NP], dlse[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int row = blk * kPrepRows + at + i * RPP;
        x[i] = y[i] = (u32x4){0, 0, 0, 0};
        lse[i] = FA_NEG_INF;
        dlse[i] = 0.f;
        if (row < p.M) {
          if (part == 0) {
            lse[i] = p.lse[b * p.sl[0] + h * p.sl[1] + row * p.sl[2]];
            if (p.dlse != nullptr) dlse[i] = p.dlse[b * p.sdl[0] + h * p.sdl[1] + row * p.sdl[2]];
          }
          x[i] = *reinterpret_cast<const u32x4*>(ob + row * p.so[2]);
          y[i] = *reinterpret_cast<const u32x4*>(gb + row * p.sdo[2]);
        }
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int row = blk * kPrepRows + at + i * RPP;
        float dot = 0.f, sq = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float y0 = DT<Tag>::to_float((uint16_t)y[i][j]), y1 = DT<Tag>::to_float((uint16_t)(y[i][j] >> 16));
          dot += DT<Tag>::to_float((uint16_t)x[i][j]) * y0;
          dot += DT<Tag>::to_float((uint16_t)(x[i][j] >> 16)) * y1;
          if constexpr (BwdTraits<Tag>::kScaled) {
            sq += y0 * y0;
            sq += y1 * y1;
          }
        }
#pragma unroll
        for (int s = 1; s < LPR; s *= 2) {
          dot += __shfl_xor(dot, s, 64);
          if constexpr (BwdTraits<Tag>::kScaled) sq += __shfl_xor(sq, s, 64);
        }
        if (part == 0) {
          const bool live = lse[i] != FA_NEG_INF;  // a row without P takes nothing from its O, dlse and bounds
          dot = live ? dot - dlse[i] : 0.f;
          float* nd = p.nd + nd_index(p, bh, row);
          nd[0] = live ? BwdTraits<Tag>::kPBias - lse[i] * 1.4426950408889634f : FA_NEG_INF;
          nd[32] = -dot;
          if (live && (__float_as_uint(sq) & 0x7fffffffu) < 0x7f800000u) top = fmaxf(top, sq);
          if ((__float_as_uint(dot) & 0x7fffffffu) < 0x7f800000u) topd = fmaxf(topd, fabsf(dot));
        }
      }
    }
  } else {
    const uint32_t v = id - nq, bh = v / (uint32_t)p.vblocks;
    const int blk = (int)(v % (uint32_t)p.vblocks), b = (int)(bh / (uint32_t)p.Hkv), h = (int)(bh % (uint32_t)p.Hkv);
    const uint16_t* vb = p.v + b * p.sv[0] + h * p.sv[1] + part * 8;
#pragma unroll 1
    for (int at = r0; at < kPrepRows; at += NP * RPP) {
      u32x4 x[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int row = blk * kPrepRows + at + i * RPP;
        x[i] = (u32x4){0, 0, 0, 0};
        if (row < p.N) x[i] = *reinterpret_cast<const u32x4*>(vb + row * p.sv[2]);
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        float sq = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x0 = DT<Tag>::to_float((uint16_t)x[i][j]), x1 = DT<Tag>::to_float((uint16_t)(x[i][j] >> 16));
          sq += x0 * x0;
          sq += x1 * x1;
        }
#pragma unroll
        for (int s = 1; s < LPR; s *= 2) sq += __shfl_xor(sq, s, 64);
        if ((__float_as_uint(sq) & 0x7fffffffu) < 0x7f800000u) top = fmaxf(top, sq);
      }
    }
  }
  if constexpr (BwdTraits<Tag>::kScaled) {
#pragma unroll
    for (int s = 32; s >= 1; s /= 2) {
      top = fmaxf(top, __shfl_xor(top, s, 64));
      topd = fmaxf(topd, __shfl_xor(topd, s, 64));
    }
    if (t % 64 == 0) {
      red[t / 64] = top;
      red[4 + t / 64] = topd;
    }
    __syncthreads();
    if (t == 0) {
      const float a = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      const float d = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
      if (id < nq) {
        p.bound[id] = a;
        p.bound[(int64_t)nq + id] = d;
      } else {
        p.bound[(int64_t)nq + id] = a;
      }
    }
  }
}

template <typename Tag, int D, int KT>
struct Bwd : LdsRows<D> {
  using L = LdsRows<D>;
  using L::frag;
  using L::tfrag;
  using L::swz;
  static constexpr int WAVES = 4;
  static constexpr int T = 32;                   // rows of a tile passing through LDS
  static constexpr int OWN = 16 * KT;            // rows owned per wave
  static constexpr int BLOCK = WAVES * OWN;      // rows owned per workgroup
  static constexpr int KS = D / 32;          // k = 32 steps over D
  static constexpr int DT16 = D / 16;        // 16-wide tiles over D
  static constexpr int ROWB = L::ROWB, CPR = L::CPR;
  static constexpr int TILEB = T * ROWB;
  // A ring of stages of two tiles each, then the stages' groups of row terms. A tile's loads are issued STAGES - 1
  // steps before its use; two stages measured 3% (D <= 128) and 7% (D = 256) faster than three or four.
  static constexpr int STAGES = 2;
  static constexpr int STAGEB = 2 * TILEB;
  static constexpr int TERMS = STAGES * STAGEB;
  static constexpr int SMEM = TERMS + STAGES * 256;
  static constexpr int NB = TILEB / 1024 / WAVES;  // LDS-DMA instructions of a wave per tile

  typedef DT<Tag> E;
  __device__ static inline uint32_t pack2(float x, float y) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    if constexpr (BwdTraits<Tag>::kScaled) {
      typedef _Float16 h2 __attribute__((ext_vector_type(2)));
      return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){x, y}, h2));
    } else {
      return E::pack2(x, y);
    }
  }

  // Tiles of 32 rows of one head, in order, into LDS; rows past the head's last read as zeros.
  struct Stream {
    const uint16_t* at;  // the next tile's first row
    uint32_t pitch;      // bytes of a row
    __device__ inline void init(const uint16_t* base, int64_t stride) {
      at = base;
      pitch = (uint32_t)stride * 2u;
    }
    __device__ inline void next() { at = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(at) + T * pitch); }
    // `left`: rows from the tile's first to the head's end (none when <= 0).
    __device__ inline void load(int left, uint32_t lds, int wave, uint32_t row, uint32_t chunk) const {
      constexpr int RPB = 1024 / ROWB;  // rows of a 1 KiB block
      const int rows = left < T ? left : T;
      const u32x4 rsrc = make_rsrc(at, rows <= 0 ? 0u : (uint32_t)(rows - 1) * pitch + (uint32_t)ROWB);
      const uint32_t off = (row & 31u) * (pitch & 0xffffffu);  // 24-bit product
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const uint32_t step = (uint32_t)(i * WAVES * RPB);
        buffer_load16_to_lds(rsrc, off + step * pitch + ((chunk ^ swz(row + step)) * 16u),
                             lds + (uint32_t)(wave + i * WAVES) * 1024u);
      }
    }
  };
  // The two tiles of a stage. A lane's place in the wave's first 1 KiB block is worked out anew for every stage: held
  // across the loop it is spilled (D = 128 has no register free), and a reload from scratch stalls the loads behind it.
  __device__ static inline void load_stage(const Stream& a, const Stream& b, int left, uint32_t lds, int wave, int lane) {
    asm volatile("" : "+v"(lane));
    const uint32_t row = (uint32_t)wave * (1024 / ROWB) + (uint32_t)lane / CPR, chunk = (uint32_t)lane % CPR;
    a.load(left, lds, wave, row, chunk);
    b.load(left, lds + TILEB, wave, row, chunk);
  }

  // The 32 rows' two terms (256 bytes). Every wave loads them, so that all have the same loads in flight.
  __device__ static inline void load_terms(const float* nd, bool live, uint32_t lds, int lane) {
    const u32x4 rsrc = make_rsrc(nd, live ? 256 : 0);
    const uint32_t dst = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %1\n\tbuffer_load_dword %0, %2, 0 offen lds"
                 :
                 : "v"((uint32_t)lane * 4u), "s"(dst), "s"(rsrc)
                 : "memory", "m0");
  }

  // The owned rows' fragments straight from memory, zeros past `rows`.
  __device__ static inline void load_frags(u32x4 (&f)[KT][KS], const uint16_t* base, int64_t stride, int row0, int rows,
                                           int lane) {
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      const int row = row0 + 16 * i + (lane & 15);
      const uint16_t* src = base + row * stride + 8 * (lane >> 4);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        f[i][ks] = (u32x4){0, 0, 0, 0};
        if (row < rows) f[i][ks] = *reinterpret_cast<const u32x4*>(src + 32 * ks);
      }
    }
  }

  // The largest of a term over the workgroup; `red` is LDS of the workgroup, free again on return.
  template <int N>
  __device__ static inline void block_max(float (&x)[N], float* red) {
    const int t = threadIdx.x;
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int s = 32; s >= 1; s /= 2) x[n] = fmaxf(x[n], __shfl_xor(x[n], s, 64));
      if (t % 64 == 0) red[4 * n + t / 64] = x[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = fmaxf(fmaxf(red[4 * n], red[4 * n + 1]), fmaxf(red[4 * n + 2], red[4 * n + 3]));
    __syncthreads();
  }
  // Largest |V row|^2 of the kv head's first `rows` rows.
  __device__ static inline float v_bound(const BwdParams& p, int b, int hk, int rows) {
    const float* vb = p.bound + 2 * (int64_t)p.B * p.H * p.prep_blocks + ((int64_t)b * p.Hkv + hk) * p.vblocks;
    const int n = (rows + kPrepRows - 1) / kPrepRows;
    float v2 = 0.f;
    for (int i = threadIdx.x; i < n; i += WAVES * 64) v2 = fmaxf(v2, vb[i]);
    return v2;
  }
  // Power of two above |dP - delta| <= |dO| |V| + |delta|. Not under 2^-60, which scales no product of fp16 numbers past
  // fp32 (rows without keys are not in the bounds), and under which no gradient is an fp16 number.
  __device__ static inline int exponent_above(float o2, float v2, float delta) {
    const float bound = sqrtf(o2) * sqrtf(v2) + delta;
    const int e = (int)(__float_as_uint(bound) >> 23) - 126;
    return e < -60 ? -60 : (e > 100 ? 100 : e);
  }
  // That of the rows which the keys from k0 on meet: of all query heads of the kv head, under a causal mask from row k0 on.
  __device__ static inline int scale_exponent(const BwdParams& p, int b, int hk, int k0, float* red) {
    const int64_t nq = (int64_t)p.B * p.H * p.prep_blocks;
    const int skip = p.causal ? k0 / kPrepRows : 0;
    float x[3] = {0.f, 0.f, v_bound(p, b, hk, p.N)};
    for (int h = 0; h < p.group; ++h) {
      const float* ob = p.bound + ((int64_t)b * p.H + (int64_t)hk * p.group + h) * p.prep_blocks;
      for (int i = skip + (int)threadIdx.x; i < p.prep_blocks; i += WAVES * 64) {
        x[0] = fmaxf(x[0], ob[i]);
        x[1] = fmaxf(x[1], ob[nq + i]);
      }
    }
    block_max(x, red);
    return uniform(exponent_above(x[0], x[2], x[1]));
  }
  __device__ static inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
  __device__ static inline float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

  __device__ static void dkdv(const BwdParams& p, char* smem, int id) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    // key blocks innermost: those running together read the same query rows
    const int nb = uniform(id % p.nblocks), part = uniform(id / p.nblocks % p.kv_splits);
    const int hkb = uniform(id / p.nblocks / p.kv_splits);
    const int b = uniform(hkb / p.Hkv), hk = uniform(hkb % p.Hkv);
    const int k0 = nb * BLOCK, kw = k0 + OWN * wave;  // first key of the block, of the wave
    float sc = 1.f, unscale = 1.f;
    if constexpr (BwdTraits<Tag>::kScaled) {
      const int e = scale_exponent(p, b, hk, k0, reinterpret_cast<float*>(smem));
      sc = pow2(-e);
      unscale = pow2(e);
    }
    u32x4 kf[KT][KS], vf[KT][KS];
    load_frags(kf, p.k + b * p.sk[0] + hk * p.sk[1], p.sk[2], kw, p.N, lane);
    load_frags(vf, p.v + b * p.sv[0] + hk * p.sv[1], p.sv[2], kw, p.N, lane);
    floatx4 dk[DT16][KT], dv[DT16][KT];
#pragma unroll
    for (int d = 0; d < DT16; ++d)
#pragma unroll
      for (int i = 0; i < KT; ++i) dk[d][i] = dv[d][i] = (floatx4){0.f, 0.f, 0.f, 0.f};

    const uint32_t lds = lds_address(smem);
    const uint32_t ro = L::row_off(lane), to = L::tr_off(lane);
    const int qt_all = (p.M + T - 1) / T;
    const int qt0 = p.causal ? k0 / T : 0;  // rows above the block's first key see none of its keys
    const int per_head = qt_all > qt0 ? qt_all - qt0 : 0;
    // this split's share of the (query head, row tile) steps
    const int all = per_head * p.group, share = (all + p.kv_splits - 1) / p.kv_splits;
    const int first = part * share, total = first >= all ? 0 : (all - first < share ? all - first : share);
    const int h0 = total > 0 ? uniform(first / per_head) : 0, ht0 = qt0 + first - h0 * per_head;

    const int hq = hk * p.group + h0;
    Stream sq, so;  // at the next load's tile
    sq.init(p.q + b * p.sq[0] + hq * p.sq[1] + ht0 * (T * p.sq[2]), p.sq[2]);
    so.init(p.dout + b * p.sdo[0] + hq * p.sdo[1] + ht0 * (T * p.sdo[2]), p.sdo[2]);
    const float* nh = p.nd + (((int64_t)b * p.H + hq) * p.row_groups + ht0) * 64;
    // from a head's end to the next head's first tile
    const int64_t skip_q = p.sq[1] - (int64_t)(per_head * T) * p.sq[2], skip_o = p.sdo[1] - (int64_t)(per_head * T) * p.sdo[2];
    const int skip_n = (p.row_groups - per_head) * 64;
    int left = p.M - ht0 * T, ahead = total;  // rows of the head, tiles of the split that are still to be loaded
    // Behind the last step the loads go on with nothing in range: the waits count on a fixed number in flight.
    auto load_next = [&](uint32_t step) {
      const uint32_t dst = lds + (uint32_t)((step % STAGES) * STAGEB);
      const int rows = ahead > 0 ? left : 0;
      load_stage(sq, so, rows, dst, wave, lane);
      load_terms(nh, rows > 0, lds + (uint32_t)(TERMS + (step % STAGES) * 256), lane);
      --ahead;
      left -= T;
      sq.next();
      so.next();
      nh += 64;
      if (left <= 0) {
        left = p.M - qt0 * T;
        sq.at += skip_q;
        so.at += skip_o;
        nh += skip_n;
      }
    };
    if (total > 0)
      for (int i = 0; i < STAGES - 1; ++i) load_next(i);
    int it = 0, ct = ht0;
    auto step = [&](auto edge_tile) {
      constexpr bool EDGE = decltype(edge_tile)::value;
      wait_vm_lds_barrier<(STAGES - 2) * (2 * NB + 1)>();
      load_next(it + STAGES - 1);
      const uint32_t rows = ro + ((uint32_t)it % STAGES) * STAGEB, cols = to + ((uint32_t)it % STAGES) * STAGEB;
      const float* nd = reinterpret_cast<const float*>(smem + TERMS + ((uint32_t)it % STAGES) * 256);
      const int q0 = ct * T;
      ++it;
      ++ct;
      if (EDGE && q0 + T - 1 < kw) return;
      u32x4 pb[KT], sb[KT];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const floatx4 nl = *reinterpret_cast<const floatx4*>(nd + 16 * i + 4 * g);
        const floatx4 nd1 = *reinterpret_cast<const floatx4*>(nd + 32 + 16 * i + 4 * g);
        floatx4 s[KT], dp[KT];
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          s[j] = (floatx4){0.f, 0.f, 0.f, 0.f};
          dp[j] = nd1;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4 a = frag(smem, rows ^ (ks << 6), i * 16 * ROWB);
          const u32x4 o = frag(smem, rows ^ (ks << 6), i * 16 * ROWB + TILEB);
#pragma unroll
          for (int j = 0; j < KT; ++j) {
            s[j] = E::mfma16(a, kf[j][ks], s[j]);
            dp[j] = E::mfma16(o, vf[j][ks], dp[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < KT; ++j) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float x = fmaf(p.c, s[j][r], nl[r]);
            if (EDGE && kw + 16 * j + c16 > q0 + 16 * i + 4 * g + r) x = FA_NEG_INF;
            s[j][r] = fast_exp2(x);
            dp[j][r] = BwdTraits<Tag>::kScaled ? s[j][r] * (dp[j][r] * sc) : s[j][r] * dp[j][r];
          }
          pb[j][2 * i] = pack2(s[j][0], s[j][1]);
          pb[j][2 * i + 1] = pack2(s[j][2], s[j][3]);
          sb[j][2 * i] = pack2(dp[j][0], dp[j][1]);
          sb[j][2 * i + 1] = pack2(dp[j][2], dp[j][3]);
        }
      }
      // a wave in its second products goes before one in its softmax (the two share a SIMD): 6% at D = 256
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int d = 0; d < DT16; ++d) {
        const u32x4 ot = tfrag(smem, cols ^ (d << 5), TILEB);
        const u32x4 qt = tfrag(smem, cols ^ (d << 5), 0);
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          dv[d][j] = E::mfma16(ot, pb[j], dv[d][j]);
          dk[d][j] = E::mfma16(qt, sb[j], dk[d][j]);
        }
      }
      __builtin_amdgcn_s_setprio(0);
    };
    // head by head: first the tiles on the diagonal, then those that all the block's keys precede
    while (it < total) {
      const int left = total - it, edge_end = p.causal ? qt0 + BLOCK / T : 0;
      for (int n = ct < edge_end ? (left < edge_end - ct ? left : edge_end - ct) : 0; n > 0 && ct < qt_all; --n)
        step(std::true_type{});
      for (int n = total - it < qt_all - ct ? total - it : qt_all - ct; n > 0; --n) step(std::false_type{});
      ct = qt0;
    }
    int key0 = threadIdx.x & 15;  // worked out anew: held through the loops it costs D = 256 a spilled fragment
    asm volatile("" : "+v"(key0));
    key0 += kw;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may reach LDS after the workgroup's end
    const float fk = p.scale * unscale * BwdTraits<Tag>::kPUnscale, fv = BwdTraits<Tag>::kPUnscale;
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      const int key = key0 + 16 * j;
      if (key >= p.N) continue;
      if (p.kv_splits > 1) {
        const int64_t w = ((int64_t)(part * p.B + b) * p.Hkv + hk) * p.N + key;
#pragma unroll
        for (int d = 0; d < DT16; ++d) {
          *reinterpret_cast<floatx4*>(p.ws_dk + w * D + 16 * d + 4 * g) = dk[d][j] * fk;
          *reinterpret_cast<floatx4*>(p.ws_dv + w * D + 16 * d + 4 * g) = dv[d][j] * fv;
        }
        continue;
      }
      uint16_t* ok = p.dk + b * p.sdk[0] + hk * p.sdk[1] + key * p.sdk[2] + 4 * g;
      uint16_t* ov = p.dv + b * p.sdv[0] + hk * p.sdv[1] + key * p.sdv[2] + 4 * g;
#pragma unroll
      for (int d = 0; d < DT16; ++d) {
        const floatx4 a = dk[d][j] * fk, v = dv[d][j] * fv;
        *reinterpret_cast<u32x2*>(ok + 16 * d) = (u32x2){pack2(a[0], a[1]), pack2(a[2], a[3])};
        *reinterpret_cast<u32x2*>(ov + 16 * d) = (u32x2){pack2(v[0], v[1]), pack2(v[2], v[3])};
      }
    }
  }

  __device__ static void dq(const BwdParams& p, char* smem, int id) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c16 = lane & 15, g = lane >> 4;
    const int at = id % p.mblocks, part = uniform(id / p.mblocks % p.q_splits);
    const int bh = uniform(id / p.mblocks / p.q_splits);
    const int mb = uniform(p.causal ? p.mblocks - 1 - at : at);  // causal: the block with the most keys first
    const int b = uniform(bh / p.H), h = uniform(bh % p.H), hk = uniform(h / p.group);
    const int m0 = mb * BLOCK, mw = m0 + OWN * wave;
    const int n_end = p.causal && m0 + BLOCK < p.N ? m0 + BLOCK : p.N;
    float v2[1] = {0.f};
    if constexpr (BwdTraits<Tag>::kScaled) {
      v2[0] = v_bound(p, b, hk, n_end);
      block_max(v2, reinterpret_cast<float*>(smem));
    }
    u32x4 qf[KT][KS], of[KT][KS];
    load_frags(qf, p.q + b * p.sq[0] + h * p.sq[1], p.sq[2], mw, p.M, lane);
    load_frags(of, p.dout + b * p.sdo[0] + h * p.sdo[1], p.sdo[2], mw, p.M, lane);
    float nl[KT], nd[KT];
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      const int row = mw + 16 * i + c16;
      nl[i] = FA_NEG_INF;
      nd[i] = 0.f;
      if (row < p.M) {
        const float* src = p.nd + nd_index(p, bh, row);
        nl[i] = src[0];
        nd[i] = src[32];
      }
    }
    // a lane's products are all of its own row: the row's own scale
    float sc[KT];
    if constexpr (BwdTraits<Tag>::kScaled) {
#pragma unroll
      for (int i = 0; i < KT; ++i) {
        float o2 = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float a = E::to_float((uint16_t)of[i][ks][j]), c = E::to_float((uint16_t)(of[i][ks][j] >> 16));
            o2 += a * a;
            o2 += c * c;
          }
        sc[i] = pow2(-exponent_above(xquad_sum(o2), v2[0], fabsf(nd[i])));
      }
    }
    floatx4 acc[DT16][KT];
#pragma unroll
    for (int d = 0; d < DT16; ++d)
#pragma unroll
      for (int i = 0; i < KT; ++i) acc[d][i] = (floatx4){0.f, 0.f, 0.f, 0.f};
    const uint32_t lds = lds_address(smem);
    const uint32_t ro = L::row_off(lane), to = L::tr_off(lane);
    const int all = (n_end + T - 1) / T, share = (all + p.q_splits - 1) / p.q_splits;
    const int first = part * share, tiles = first >= all ? first : (all - first < share ? all : first + share);
    Stream sk, sv;
    sk.init(p.k + b * p.sk[0] + hk * p.sk[1] + first * (T * p.sk[2]), p.sk[2]);
    sv.init(p.v + b * p.sv[0] + hk * p.sv[1] + first * (T * p.sv[2]), p.sv[2]);
    // rows that are still to be loaded: past the split's last tile none are
    int left = (tiles * T < p.N ? tiles * T : p.N) - first * T;
    auto load = [&](uint32_t t) {
      const uint32_t dst = lds + (uint32_t)((t % STAGES) * STAGEB);
      load_stage(sk, sv, left, dst, wave, lane);
      left -= T;
      sk.next();
      sv.next();
    };
    if (first < tiles)
      for (int i = 0; i < STAGES - 1; ++i) load(first + i);
    auto step = [&](int t, auto edge_tile) {
      constexpr bool EDGE = decltype(edge_tile)::value;
      wait_vm_lds_barrier<(STAGES - 2) * 2 * NB>();
      load(t + STAGES - 1);
      const uint32_t rows = ro + ((uint32_t)t % STAGES) * STAGEB, cols = to + ((uint32_t)t % STAGES) * STAGEB;
      const int n0 = t * T;
      if (EDGE && p.causal && n0 > mw + OWN - 1) return;
      u32x4 sb[KT];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        floatx4 s[KT], dp[KT];
#pragma unroll
        for (int j = 0; j < KT; ++j) {
          s[j] = (floatx4){0.f, 0.f, 0.f, 0.f};
          dp[j] = (floatx4){nd[j], nd[j], nd[j], nd[j]};
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const u32x4 a = frag(smem, rows ^ (ks << 6), i * 16 * ROWB);
          const u32x4 v = frag(smem, rows ^ (ks << 6), i * 16 * ROWB + TILEB);
#pragma unroll
          for (int j = 0; j < KT; ++j) {
            s[j] = E::mfma16(a, qf[j][ks], s[j]);
            dp[j] = E::mfma16(v, of[j][ks], dp[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < KT; ++j) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float x = fmaf(p.c, s[j][r], nl[j]);
            if (EDGE) {
              const int key = n0 + 16 * i + 4 * g + r;
              if (key >= p.N || (p.causal && key > mw + 16 * j + c16)) x = FA_NEG_INF;
            }
            const float e = fast_exp2(x);
            dp[j][r] = BwdTraits<Tag>::kScaled ? e * (dp[j][r] * sc[j]) : e * dp[j][r];
          }
          sb[j][2 * i] = pack2(dp[j][0], dp[j][1]);
          sb[j][2 * i + 1] = pack2(dp[j][2], dp[j][3]);
        }
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int d = 0; d < DT16; ++d) {
        const u32x4 kt = tfrag(smem, cols ^ (d << 5), 0);
#pragma unroll
        for (int j = 0; j < KT; ++j) acc[d][j] = E::mfma16(kt, sb[j], acc[d][j]);
      }
      __builtin_amdgcn_s_setprio(0);
    };
    // whole tiles before the block's first row, then those on the diagonal or past the last key
    const int whole = p.causal && m0 < p.N ? m0 / T : p.N / T;
    int t = first;
    for (; t < tiles && t < whole; ++t) step(t, std::false_type{});
    for (; t < tiles; ++t) step(t, std::true_type{});
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int j = 0; j < KT; ++j) {
      const int row = mw + 16 * j + c16;
      if (row >= p.M) continue;
      const float f = p.scale * (BwdTraits<Tag>::kScaled ? BwdTraits<Tag>::kPUnscale / sc[j] : 1.f);
      if (p.q_splits > 1) {
        const int64_t w = ((int64_t)(part * p.B + b) * p.H + h) * p.M + row;
#pragma unroll
        for (int d = 0; d < DT16; ++d) *reinterpret_cast<floatx4*>(p.ws_dq + w * D + 16 * d + 4 * g) = acc[d][j] * f;
        continue;
      }
      uint16_t* out = p.dq + b * p.sdq[0] + h * p.sdq[1] + row * p.sdq[2] + 4 * g;
#pragma unroll
      for (int d = 0; d < DT16; ++d) {
        const floatx4 a = acc[d][j] * f;
        *reinterpret_cast<u32x2*>(out + 16 * d) = (u32x2){pack2(a[0], a[1]), pack2(a[2], a[3])};
      }
    }
  }
};

// dK/dV blocks first (they are the longer ones), then dQ blocks, in one grid, each kind in runs that keep a head's
// blocks on one XCD. Grids small enough to be split alternate the two kinds in proportion instead: the working
// set fits the L2 either way, and blocks of unlike lengths run side by side (bf16 B1 12/2 heads N4096 D128 causal
// 298 -> 272 us; large grids lose 3 to 5% by it, for L2 misses).
template <typename Tag, int D, int KT, int PER_CU>
__global__ __launch_bounds__(256, PER_CU) void fa_bwd_kernel(BwdParams p) {
  __shared__ __align__(1024) char smem[Bwd<Tag, D, KT>::SMEM];
  const uint32_t id = blockIdx.x;
  bool is_kv = id < (uint32_t)p.kv_total;
  int block = is_kv ? xcd_remap(id, p.kv_total) : xcd_remap(id - p.kv_total, p.q_total);
  if (p.kv_splits * p.q_splits > 1 && p.kv_total % 8 == 0 && p.q_total % 8 == 0) {
    const uint32_t kv = (uint32_t)p.kv_total / 8, q = (uint32_t)p.q_total / 8, xcd = id % 8, slot = id / 8;
    const uint32_t before = (uint32_t)((uint64_t)slot * kv / (kv + q));  // dK/dV blocks of the XCD ahead of this slot
    is_kv = (uint32_t)((uint64_t)(slot + 1) * kv / (kv + q)) > before;
    block = is_kv ? xcd * kv + before : xcd * q + (slot - before);
  }
  block = __builtin_amdgcn_readfirstlane(block);
  if (is_kv)
    Bwd<Tag, D, KT>::dkdv(p, smem, block);
  else
    Bwd<Tag, D, KT>::dq(p, smem, block);
}

// Sums of the splits' partial gradients, in split order: a thread takes four channels of one row. Bound by memory:
// ten partials of 2 x 4 MB in 15 us (bf16 B1 12/2 heads N4096 causal).
template <typename Tag, int D>
__global__ __launch_bounds__(256) void fa_bwd_reduce_kernel(BwdParams p) {
  const int64_t kv_rows = p.kv_splits > 1 ? (int64_t)p.B * p.Hkv * p.N : 0;
  const int64_t q_rows = p.q_splits > 1 ? (int64_t)p.B * p.H * p.M : 0;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int64_t row = id / (D / 4);
  const int d = (int)(id % (D / 4)) * 4;
  if (row >= 2 * kv_rows + q_rows) return;
  const float* src;
  uint16_t* out;
  const int64_t* st;
  int64_t rows;
  int splits, heads, len;
  if (row < 2 * kv_rows) {
    const bool second = row >= kv_rows;
    row -= second ? kv_rows : 0;
    src = second ? p.ws_dv : p.ws_dk;
    out = second ? p.dv : p.dk;
    st = second ? p.sdv : p.sdk;
    rows = kv_rows, splits = p.kv_splits, heads = p.Hkv, len = p.N;
  } else {
    row -= 2 * kv_rows;
    src = p.ws_dq;
    out = p.dq;
    st = p.sdq;
    rows = q_rows, splits = p.q_splits, heads = p.H, len = p.M;
  }
  floatx4 sum = *reinterpret_cast<const floatx4*>(src + row * D + d);
  for (int i = 1; i < splits; ++i) sum += *reinterpret_cast<const floatx4*>(src + (i * rows + row) * D + d);
  const int64_t bh = row / len;
  out += bh / heads * st[0] + bh % heads * st[1] + row % len * st[2] + d;
  *reinterpret_cast<u32x2*>(out) = (u32x2){DT<Tag>::pack2(sum[0], sum[1]), DT<Tag>::pack2(sum[2], sum[3])};
}

#define FA_BWD_ENTRY(TAG, DTYPE, D, KT, PER_CU)                                                          \
  {DTYPE, D, (const void*)&fa_bwd_prep_kernel<TAG, D>, (const void*)&fa_bwd_kernel<TAG, D, KT, PER_CU>, \
   (const void*)&fa_bwd_reduce_kernel<TAG, D>, Bwd<TAG, D, KT>::BLOCK, kPrepRows, PER_CU}

static const BwdKernelEntry kBwdEntries[] = {
    FA_BWD_ENTRY(f16_t, FA_DTYPE_F16, 64, 2, 2),
    FA_BWD_ENTRY(f16_t, FA_DTYPE_F16, 128, 2, 2),
    FA_BWD_ENTRY(f16_t, FA_DTYPE_F16, 256, 2, 1),
    FA_BWD_ENTRY(bf16_t, FA_DTYPE_BF16, 64, 2, 2),
    FA_BWD_ENTRY(bf16_t, FA_DTYPE_BF16, 128, 2, 2),
    FA_BWD_ENTRY(bf16_t, FA_DTYPE_BF16, 256, 2, 1),
};

const BwdKernelEntry* fa_bwd_registry(int* count) {
  *count = (int)(sizeof(kBwdEntries) / sizeof(kBwdEntries[0]));
  return kBwdEntries;
}

}  // namespace fa
