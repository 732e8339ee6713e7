// Softmax cross entropy of a linear vocabulary head without its logits, and its gradient, on the 5th-generation
// tensor cores (sm_100a).
//
//   z[i][v] = sum_k h[i][k] w[v][k] + b[v],   loss[i] = log sum_v exp z[i][v] - z[i][label_i]
//   g[i][v] = c_i (exp(z[i][v] - lse_i) - [v = label_i]),   dh = g w,   dw = g^T h,   db[v] = sum_i g[i][v]
//
// with c_i the weight of row i in the reduced loss (0 for an ignored row).
//
// Loss: one tensor-core product whose epilogue reduces each 128-column slice of a row to (maximum, sum of
// exponentials) in 32 bits while the accumulator is in tensor memory; the logits never reach memory.
// xent_finish_kernel joins a row's slices. Bound by the product: 2 rows vocab hidden operations.
// Gradient: rows go through in chunks (all of them in one, unless 16 bits x rows x vocab pass the chunk limit). The same
// product also leaves e = exp(z - slice maximum), rounded to the operands' 16-bit type, in the workspace;
// once a row's sum is known xent_rescale_kernel turns e into g in place (one read and one write of 16 bits per
// logit: 4 bytes against 6 hidden operations), and two more products read g: dh directly, dw with both
// operands taken along their non-contiguous direction (MN-major tiles), so nothing is transposed in memory.
// Keeping e for a chunk of rows costs its two passes; recomputing the logits instead would cost a
// fourth product of the size of the other three.
// g is rounded to 16 bits twice (e, then g: at most half a step each), sums are 32-bit throughout. For fp16 both
// carry a factor 2^15 (their values lie in [-1, 1], most of them far below fp16's smallest normal number).
//
// The product kernel is persistent, a CTA pair per 256 x 256 tile (cta_group::2): warp 0 feeds a six-stage ring
// by TMA, one thread of the leader issues tcgen05.mma into one of two 256-column accumulators, eight warps
// empty the other one. All waits are bounded; a wait that gives up sets the status word and every role leaves. While the
// word is set losses and gradients come out as NaN.
//
// Measured (bf16, device time): loss of 2,048 x 2,048 x 32,768 187 us = 1,470 TFLOP/s, of 16,384 x 4,096 x 131,072 13.4 ms =
// 1,315 TFLOP/s under the power cap; with gradients 600 to 690 us and (8,192 rows) 20.8 to 21.8 ms. The tensor pipe is busy 78 % of the
// logits product (its shared memory is: 64 KB of tiles written and as much read per 512 tensor cycles and SM) and
// 94 % of the gradient products; the rescaling pass is 3 % (4,096 features) to 9 % (2,048) of a step.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include <atomic>

#include "sm100.cuh"
#include "xent.cuh"

namespace evox {
namespace {

constexpr int TM = 256, TN = 256, BK = 64, STAGES = 6;  // one tile of a CTA pair; each CTA holds half of both operands
constexpr int kThreads = 64 + 256;
constexpr int kChunkBlocks = 16;  // blocks of the reduction per accumulator of a logit
constexpr uint32_t kOperandBytes = 128 * BK * 2;
constexpr uint32_t kStageBytes = 2 * kOperandBytes;
// half of a warp's 32 x 128 results on its way out: a swizzled tile of 32 rows x 128 bytes
constexpr uint32_t kOffOut = STAGES * kStageBytes;
constexpr uint32_t kOutBytes = 32 * 64 * 2;
constexpr uint32_t kOffBars = kOffOut + 8 * kOutBytes;
constexpr uint32_t kSmemBytes = kOffBars + 256;  // 229,632 B of the 232,448 B a CTA may use

// What the epilogue leaves: kLoss the softmax statistics, kProb the exponentials too, kProbLow also what their rounding to
// 16 bits left, kOut the product itself.
enum { kLoss = 0, kProb = 1, kOut = 2, kProbLow = 3 };

// One product D = A B^T over the reduction index, as tiles of 256 x 256.
struct Product {
  long long M, N;
  int k_blocks;            // of BK
  int splits;              // the reduction is divided among this many work items per tile (kOut)
  int tiles_m, tiles_n;
  int m_fast, group;       // tiles run through `group` of the one direction, then all of the other
  uint32_t idesc;
  int a_mn;                // A is contiguous along its own rows instead of the reduction (kOut)
  // kOut: D, scaled
  void* out16;             // [M][N], 16 bits, dense (final), or null
  float* out32;            // [splits][M][ld32] partial sums, or the running sum over row chunks, or null
  long long ld32;
  int tiled_out;           // out16 has a tensor map (rows on 16-byte boundaries)
  int add32;               // add what out32 holds before storing (or to out16)
};
// kOut does two products in one launch, dh and dw, so that neither waits for the other's last tiles: CTA pair q takes items
// q, q + pairs, ... of the first, then some of the second's: the first `heavy` pairs, which have one item more of the first
// product, `per_heavy` of them, the others `early` more before that. Neighbouring items run at the same time, so
// that the operand lines they share are read from memory once.
struct ProductArgs {
  Product p[2];
  int pairs, heavy, items[2], per_heavy, early;
  int chunks;              // accumulators that a tile's reduction is divided among (all but kOut)
  uint32_t stage_bytes;    // what the copies of a stage bring to both CTAs
  int* error_flag;
  const float* scale;      // device scalar (kOut)
  // all but kOut
  const float* bias;       // [N] or null
  const long long* labels; // [M]
  float2* stats;           // [slices][ld_stats]: (maximum, sum of exponentials)
  long long ld_stats;
  float* label_logit;      // [M]
};
struct Maps {
  CUtensorMap a[2], b[2], out[2];  // of the two products; of kProb and kProbLow: out = e and what its rounding left
};

template <bool FP16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (FP16) {
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  } else {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
}
template <bool FP16>
__device__ __forceinline__ unsigned short pack1(float a) {
  if constexpr (FP16) return __half_as_ushort(__float2half_rn(a));
  else return __bfloat16_as_ushort(__float2bfloat16_rn(a));
}
template <bool FP16>
__device__ __forceinline__ float2 unpack2(uint32_t p) {
  if constexpr (FP16) return __half22float2(*reinterpret_cast<const __half2*>(&p));
  else return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
}
template <bool FP16>
constexpr float kProbScale = FP16 ? 32768.0f : 1.0f;

// 32 bytes to an aligned place.
__device__ __forceinline__ void store_32_bytes(float* to, const float (&p)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "f"(p[0]), "f"(p[1]), "f"(p[2]), "f"(p[3]),
               "f"(p[4]), "f"(p[5]), "f"(p[6]), "f"(p[7])
               : "memory");
}

// Place of 16-byte piece `piece` (0..7) of row `row` (0..31) in a warp's outgoing tile of 128-byte rows, with the 128-byte
// swizzle of its tensor map; neighbouring rows' pieces fall into different banks.
__device__ __forceinline__ uint32_t out_place(int row, int piece) { return (uint32_t)(row * 128 + ((piece ^ (row & 7)) << 4)); }
// This thread's row (64 values, scaled) into the warp's outgoing tile. LOW: z becomes what the rounding left.
template <bool FP16, bool LOW = false>
__device__ __forceinline__ void put_row(uint8_t* out, int lane, float (&za)[32], float (&zb)[32], float scale) {
#pragma unroll
  for (int j = 0; j < 64; j += 8) {
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float &a = j < 32 ? za[j + 2 * i] : zb[j - 32 + 2 * i], &b = j < 32 ? za[j + 2 * i + 1] : zb[j - 32 + 2 * i + 1];
      p[i] = pack2<FP16>(a * scale, b * scale);
      if constexpr (LOW) {
        const float2 kept = unpack2<FP16>(p[i]);
        a = fmaf(a, scale, -kept.x);
        b = fmaf(b, scale, -kept.y);
      }
    }
    *reinterpret_cast<uint4*>(out + out_place(lane, j / 8)) = make_uint4(p[0], p[1], p[2], p[3]);
  }
}
// The warp's tile to rows from `row` on and columns from `col` on of the map's matrix, which cuts off what lies outside.
__device__ __forceinline__ void send_rows(const CUtensorMap* map, uint8_t* out, int lane, int col, int row) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"((unsigned long long)map),
                 "r"(smem_u32(out)), "r"(col), "r"(row)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}
// Until the copy that was sent has read the warp's tile.
__device__ __forceinline__ void wait_sent(int lane) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
}


// Operand descriptor of an MN-major tile: 64 elements of the row direction are contiguous (128 bytes, swizzled), one
// such line per reduction index; 8 lines make 1,024 bytes, the next 64 row elements start 64 lines further.
__device__ __forceinline__ unsigned long long umma_desc_mn(uint32_t smem_addr) {
  return umma_desc(smem_addr) | ((unsigned long long)((64u * 128u) >> 4) << 16);
}

struct Item {
  int which;               // product
  int m, n;                // tile
  int split, kb0, kb1;     // blocks of the reduction
};
// In 32 bits (the host refuses more work items): one thread computes this between two tiles' instructions.
__device__ __forceinline__ Item item_of(const Product& a, int which, unsigned work) {
  const unsigned tiles = (unsigned)a.tiles_m * (unsigned)a.tiles_n;
  Item t;
  t.which = which;
  unsigned r = work;
  t.split = 0;
  t.kb0 = 0;
  t.kb1 = a.k_blocks;
  if (a.splits > 1) {
    t.split = (int)(work / tiles);
    r = work - (unsigned)t.split * tiles;
    const unsigned each = (unsigned)a.k_blocks / (unsigned)a.splits, more = (unsigned)a.k_blocks - each * (unsigned)a.splits;
    t.kb0 = (int)(t.split * each + min((unsigned)t.split, more));  // the first `more` splits have a block more
    t.kb1 = t.kb0 + (int)(each + ((unsigned)t.split < more ? 1u : 0u));
  }
  const unsigned fast = a.m_fast ? a.tiles_m : a.tiles_n, slow = a.m_fast ? a.tiles_n : a.tiles_m;
  const unsigned first = r / ((unsigned)a.group * slow) * (unsigned)a.group;
  const unsigned width = min((unsigned)a.group, fast - first);
  const unsigned q = r - first * slow, s = q / width, f = first + (q - s * width);
  t.m = (int)(a.m_fast ? f : s);
  t.n = (int)(a.m_fast ? s : f);
  return t;
}

// The products of ProductArgs; in kOut B is contiguous along its own rows, elsewhere both operands along the reduction.
template <int MODE, bool FP16>
__global__ void __launch_bounds__(kThreads, 1) xent_product_kernel(const __grid_constant__ Maps maps, const ProductArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem_base = smem_u32(smem_raw);
  if ((smem_base & 1023u) != 0) {  // the swizzled tiles need a 1024-byte aligned window: refuse to run otherwise
    overlapped_start();
    if (threadIdx.x == 0) atomicCAS(a.error_flag, 0, 5);
    return;
  }
  const uint32_t bars = smem_base + kOffBars;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (STAGES + s); };
  auto tfull_bar = [&](int b) { return bars + 8u * (2 * STAGES + b); };
  auto tempty_bar = [&](int b) { return bars + 8u * (2 * STAGES + 2 + b); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_raw + kOffBars + 8 * (2 * STAGES + 4));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta_rank = cluster_rank();
  // this pair's work: `count0` items of the first product, then `count1` of the second
  const int pair = blockIdx.x >> 1;
  const int count0 = a.items[0] > pair ? (a.items[0] - pair - 1) / a.pairs + 1 : 0;
  const int early = pair < a.heavy ? 0 : a.early;
  auto second = [&](int j) {  // its j-th item of the second product
    if (j < early) return j * (a.pairs - a.heavy) + pair - a.heavy;
    return a.early * (a.pairs - a.heavy) + (j - early) * a.pairs + pair;
  };
  int count1 = MODE == kOut ? early + a.per_heavy : 0;
  while (count1 > 0 && second(count1 - 1) >= a.items[1]) --count1;
  const int n_items = count0 + count1;
  auto item = [&](int i) {
    if (MODE != kOut || i < count0) return item_of(a.p[0], 0, (unsigned)(pair + i * a.pairs));
    return item_of(a.p[1], 1, (unsigned)second(i - count0));
  };
  const int chunks = MODE == kOut ? 1 : a.chunks;  // a tile's reduction goes through these accumulators one after the other

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), 2 * 8);  // the leader's collects both epilogues, an arrival per warp
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers exist before anything is sent to them
  fence_after_sync();
  const uint32_t tmem_base = *((volatile uint32_t*)tmem_slot);
  overlapped_start();  // nothing of global memory was touched so far

  if (warp == 0) {
    // ------------------------------- TMA producer ------------------------------------------
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t leader_full0 = map_to_cta(full_bar(0), 0u);
      for (int i = 0; i < n_items && ok; ++i) {
        const Item t = item(i);
        const int m0 = t.m * TM + (int)cta_rank * 128, n0 = t.n * TN + (int)cta_rank * 128;
        const bool a_mn = MODE == kOut && a.p[t.which].a_mn;
        const CUtensorMap *map_a = &maps.a[t.which], *map_b = &maps.b[t.which];
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, a.error_flag, 1)) {
            ok = false;
            break;
          }
          if (cta_rank == 0) mbar_expect_tx(full_bar(s), a.stage_bytes);
          const uint32_t fb = leader_full0 + 8u * s, sa = smem_base + s * kStageBytes, sb = sa + kOperandBytes;
          const int k0 = kb * BK;
          if (a_mn) {
            tma_load_2d_pair(sa, map_a, fb, m0, k0);
            tma_load_2d_pair(sa + kOperandBytes / 2, map_a, fb, m0 + 64, k0);
          } else if (cta_rank == 0 || a.stage_bytes == 2 * kStageBytes) {
            tma_load_2d_pair(sa, map_a, fb, k0, m0);
          }
          if constexpr (MODE == kOut) {
            tma_load_2d_pair(sb, map_b, fb, n0, k0);
            tma_load_2d_pair(sb + kOperandBytes / 2, map_b, fb, n0 + 64, k0);
          } else {
            tma_load_2d_pair(sb, map_b, fb, k0, n0);
          }
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // the leader's releases of this CTA's stages arrive asynchronously: see the last one of every stage land
      // before this CTA may leave
      for (int q = 0; q < STAGES && ok; ++q) {
        if (!mbar_wait(empty_bar(s), ph ^ 1u, a.error_flag, 1)) ok = false;
        if (++s == STAGES) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (!ok) settle();
    }
  } else if (warp == 1) {
    // ------------------------------- MMA issuer --------------------------------------------
    if (lane == 0 && cta_rank == 0) {
      int s = 0;
      uint32_t ph = 0;
      long long it = 0;
      bool ok = true;
      Item next = item(0);
      for (int i = 0; i < n_items && ok; ++i) {
        const Item t = next;
        const bool a_mn = MODE == kOut && a.p[t.which].a_mn;
        const uint32_t idesc = a.p[t.which].idesc;
        for (int chunk = 0; chunk < chunks && ok; ++chunk, ++it) {
          const int kb0 = t.kb0 + chunk * kChunkBlocks, kb1 = chunk + 1 < chunks ? kb0 + kChunkBlocks : t.kb1;
          const int buf = (int)(it & 1);
          if (!mbar_wait(tempty_bar(buf), (uint32_t)((it >> 1) & 1) ^ 1u, a.error_flag, 2)) {
            ok = false;
            break;
          }
          fence_after_sync();
          const uint32_t d_tmem = tmem_base + (uint32_t)(buf * TN);
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(full_bar(s), ph, a.error_flag, 3)) {
              ok = false;
              break;
            }
            fence_after_sync();
            const uint32_t sa = smem_base + s * kStageBytes, sb = sa + kOperandBytes;
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
              // 16 reduction indices further: 32 bytes along a K-major line, 16 lines of an MN-major tile
              const unsigned long long da = a_mn ? umma_desc_mn(sa + k * 2048) : umma_desc(sa + k * 32);
              const unsigned long long db = MODE == kOut ? umma_desc_mn(sb + k * 2048) : umma_desc(sb + k * 32);
              umma_f16_pair(d_tmem, da, db, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
            }
            umma_commit_pair(empty_bar(s));  // stage reusable in both CTAs once these products have read it
            if (kb == t.kb0 && i + 1 < n_items) next = item(i + 1);  // while these run
            if (++s == STAGES) {
              s = 0;
              ph ^= 1u;
            }
          }
          if (ok) umma_commit_pair(tfull_bar(buf));  // accumulator complete
        }
      }
      if (!ok) settle();
    }
  } else {
    // ------------------------------- epilogue (256 threads) --------------------------------
    const int quarter = warp & 3;          // TMEM lanes this warp may read
    const int half = (warp - 2) >> 2;      // which 128 of the tile's 256 columns this warp handles
    const uint32_t leader_tempty0 = map_to_cta(tempty_bar(0), 0u);
    uint8_t* out = smem_raw + kOffOut + (warp - 2) * kOutBytes;
    long long it = 0;
    for (int i = 0; i < n_items; ++i) {
      const Item t = item(i);
      const Product& p = a.p[MODE == kOut ? t.which : 0];
      const long long row = (long long)t.m * TM + cta_rank * 128 + quarter * 32 + lane;
      const long long col0 = (long long)t.n * TN + half * kSlice;
      const bool live = row < p.M;
      const int width = (int)max(0ll, min((long long)kSlice, p.N - col0));  // columns of this slice that exist
      long long label = -1;  // column of the slice, if it is there
      if constexpr (MODE != kOut) {
        if (live) label = __ldg(a.labels + row) - col0;  // on its way while the accumulator fills
        if (label >= width) label = -1;
      }
      float z[4][32];  // this thread's row of the slice
      bool ready = true;
      for (int chunk = 0; chunk < chunks; ++chunk, ++it) {
        const int buf = (int)(it & 1);
        ready = mbar_wait(tfull_bar(buf), (uint32_t)((it >> 1) & 1), a.error_flag, 4);
        ready = __all_sync(0xffffffffu, ready);
        if (!ready) break;
        fence_after_sync();
        const uint32_t taddr = tmem_base + (uint32_t)(buf * TN + half * kSlice) + ((uint32_t)(quarter * 32) << 16);
        if (chunk == 0) {
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(taddr + c * 32, reinterpret_cast<uint32_t(&)[32]>(z[c]));
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t v[32];
            tmem_ld32(taddr + c * 32, v);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) z[c][j] += __uint_as_float(v[j]);
          }
        }
        // the accumulator is in registers: one arrival per warp hands it back. Relaxed: what goes back is tensor memory whose
        // loads are complete, and a release would make the warp wait for its stores of the previous tile
        // (ncu, 1,003 x 1,000 x 50,021: a fifth of the epilogue's stalls)
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(leader_tempty0 + 8u * buf);
      }
      if (!ready) {
        settle();
        // what this warp still had to write becomes NaN: memory that nothing wrote must not pass for a gradient. (Losses and
        // exponentials need no such care: the status word turns them into NaN when the rows are joined.)
        for (int left = i; MODE == kOut && left < n_items; ++left) {
          const Item u = item(left);
          const Product& q = a.p[u.which];
          const long long first = (long long)u.m * TM + cta_rank * 128 + quarter * 32, from = (long long)u.n * TN + half * kSlice;
          for (long long r = first; r < min(first + 32, q.M); ++r)
            for (long long c = from + lane; c < min(from + kSlice, q.N); c += 32) {
              if (q.out16) reinterpret_cast<unsigned short*>(q.out16)[r * q.N + c] = 0x7fffu;
              else q.out32[((long long)u.split * q.M + r) * q.ld32 + c] = NAN;
            }
        }
        break;
      }
      if constexpr (MODE == kOut) {
        const float scale = a.scale ? __ldg(a.scale) : 1.0f;
        float* o32 = p.out32 ? p.out32 + ((long long)t.split * p.M + row) * p.ld32 + col0 : nullptr;
        if (o32 && live) {  // rows of out32 hold a multiple of eight columns
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              if (c * 32 + j < width) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = z[c][j + i] * scale;
                if (p.add32) {
#pragma unroll
                  for (int i = 0; i < 8; ++i) v[i] += o32[c * 32 + j + i];
                }
                if (!p.out16) store_32_bytes(o32 + c * 32 + j, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) z[c][j + i] = v[i];
              }
            }
        }
        if (p.out16) {
          const long long row0 = row - lane;
          const float s16 = o32 ? 1.0f : scale;
#pragma unroll
          for (int half64 = 0; half64 < 2; ++half64) {
            if (half64 * 64 >= width || row0 >= p.M) break;
            wait_sent(lane);
            put_row<FP16>(out, lane, z[2 * half64], z[2 * half64 + 1], s16);
            if (p.tiled_out) {
              send_rows(&maps.out[t.which], out, lane, (int)col0 + half64 * 64, (int)row0);
            } else {  // rows that start anywhere: row by row, lanes along it
              __syncwarp();
              unsigned short* to = reinterpret_cast<unsigned short*>(p.out16) + row0 * p.N + col0 + half64 * 64;
              const int rows_here = (int)min(32ll, p.M - row0);
              if (p.N % 2 == 0 && (reinterpret_cast<uintptr_t>(p.out16) & 3u) == 0) {  // pairs of columns, 128 bytes of a row at once
                if (half64 * 64 + 2 * lane < width) {
#pragma unroll 8
                  for (int i = 0; i < rows_here; ++i)
                    *reinterpret_cast<uint32_t*>(to + i * p.N + 2 * lane) =
                        *reinterpret_cast<const uint32_t*>(out + out_place(i, lane >> 2) + (lane & 3) * 4);
                }
              } else {
#pragma unroll 4
                for (int i = 0; i < rows_here; ++i)
#pragma unroll
                  for (int c = lane; c < 64; c += 32)
                    if (half64 * 64 + c < width)
                      to[i * p.N + c] = *reinterpret_cast<const unsigned short*>(out + out_place(i, c >> 3) + (c & 7) * 2);
              }
            }
          }
        }
      } else {
        if (a.bias) {
          if (width == kSlice && (reinterpret_cast<uintptr_t>(a.bias) & 15u) == 0) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 b = __ldg(reinterpret_cast<const float4*>(a.bias + col0 + c * 32 + j));
                z[c][j] += b.x; z[c][j + 1] += b.y; z[c][j + 2] += b.z; z[c][j + 3] += b.w;
              }
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (c * 32 + j < width) z[c][j] += __ldg(a.bias + col0 + c * 32 + j);
          }
        }
        if (width < kSlice) {  // columns past the vocabulary
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c * 32 + j >= width) z[c][j] = -INFINITY;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) keep_label(z[c], label, c * 32, a.label_logit + row);
        float top[4], part[4];  // four chains at once
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          top[c] = z[c][0];
#pragma unroll
          for (int j = 1; j < 32; ++j) top[c] = fmaxf(top[c], z[c][j]);
        }
        const float m = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), -INFINITY);
#pragma unroll
        for (int c = 0; c < 4; ++c) exp_from(z[c], m);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          part[c] = z[c][0];
#pragma unroll
          for (int j = 1; j < 32; ++j) part[c] += z[c][j];
        }
        if (live && width > 0)
          a.stats[(long long)(t.n * 2 + half) * a.ld_stats + row] = make_float2(m, (part[0] + part[1]) + (part[2] + part[3]));
        if constexpr (MODE != kLoss) {
          const long long row0 = row - lane;
#pragma unroll
          for (int half64 = 0; half64 < 2; ++half64) {
            if (half64 * 64 >= width || row0 >= p.M) break;
            wait_sent(lane);
            put_row<FP16, MODE == kProbLow>(out, lane, z[2 * half64], z[2 * half64 + 1], kProbScale<FP16>);
            send_rows(&maps.out[0], out, lane, (int)col0 + half64 * 64, (int)row0);
            if constexpr (MODE == kProbLow) {
              wait_sent(lane);
              put_row<FP16>(out, lane, z[2 * half64], z[2 * half64 + 1], 1.0f);
              send_rows(&maps.out[1], out, lane, (int)col0 + half64 * 64, (int)row0);
            }
          }
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  // the pair leaves together: until here the peer may still arrive on this CTA's barriers, and the leader's
  // products read this CTA's shared memory
  cluster_sync_all();
  if (warp == 1) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------
// Few rows (up to 64). The product is bound by reading the weight once, so the operands change sides: 256 rows of the long
// operand (the weight's, or its columns for dh) fill the tensor core's rows and the tokens are its 32 or 64 columns. A
// block of the reduction then takes an eighth of the tensor cycles of a tile with 256 columns, and the ring holds
// nearly nothing but the weight (ten stages). Products into one accumulator follow one another at about 160 cycles
// however narrow they are, so the four of a block go to four accumulators. Accumulator lanes are weight rows, so the softmax statistics of a token
// run across lanes and the four warps that share a slice of 128. Measured: one token, 32,000 x 4,096: 54 us with the joining
// kernel (4.9 TB/s of the weight; 60.7 us as a 256 x 256 tile with one row in use). Two columns of 32 are what a stage's token
// tile holds, hence 64 rows; at that many, here and as 256 x 256 tiles (loss / gradient, us): 4,096 x 32,000 58 / 170 and 63 / 174,
// 2,048 x 131,072 102 / 328 and 116 / 329, 2,048 x 8,000 20 / 45 and 22 / 48, 256 x 1,000 10.3 / 23.1 and 10.5 / 21.5.
// ---------------------------------------------------------------------------------------------
constexpr int kFewRows = 64;
constexpr int kFewSums = BK / 16;       // accumulators at a time, one for each product of a block
constexpr int kFewChunkBlocks = 16;     // blocks of the reduction that they take before they are joined
constexpr int kFewStages = 10;
constexpr uint32_t kFewStageBytes = kOperandBytes + 32 * 128;  // 128 lines of the long operand, up to 32 tokens' of the short one
constexpr uint32_t kFewOffBars = kFewStages * kFewStageBytes;
constexpr uint32_t kFewOffShared = kFewOffBars + 256;          // float [2: maxima, sums][2 halves][4 warps][32 tokens]
constexpr uint32_t kFewSmemBytes = kFewOffShared + 2 * 2 * 4 * 32 * 4;

struct FewArgs {
  long long M;             // rows of the long operand: words, or hidden features
  int rows;                // tokens
  int k_blocks, splits, chunks, tiles;
  uint32_t idesc;
  int* error_flag;
  // all but kOut
  const float* bias;
  const long long* labels;
  float2* stats;
  long long ld_stats;
  float* label_logit;
  unsigned short* e;       // [rows][ld_e]
  unsigned short* e_low;
  long long ld_e;
  // kOut
  unsigned short* out16;   // [rows][M], or null
  float* out32;            // [splits][rows][ld32], or null
  long long ld32;
  const float* scale;
  int* tickets;            // [rows], set to 0 for the kernel that joins partial logits, or null
};

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

// Across the warp: lane l gets the maximum or the sum over all lanes of v[l % T]. Halves of the values change hands in every step,
// so T values cost T - 1 exchanges (and T more for T = 16, whose first step keeps them all).
template <int T, bool MAX>
__device__ __forceinline__ float reduce_lanes(const float (&x)[T], int lane) {
  float v[T];
#pragma unroll
  for (int j = 0; j < T; ++j) v[j] = x[j];
  auto join = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
#pragma unroll
  for (int step = 16; step >= T; step >>= 1)
#pragma unroll
    for (int j = 0; j < T; ++j) v[j] = join(v[j], __shfl_xor_sync(0xffffffffu, v[j], step));
#pragma unroll
  for (int step = T / 2; step > 0; step >>= 1) {
    const bool high = lane & step;
#pragma unroll
    for (int j = 0; j < step; ++j) {
      const float give = high ? v[j] : v[j + step], keep = high ? v[j + step] : v[j];
      v[j] = join(keep, __shfl_xor_sync(0xffffffffu, give, step));
    }
  }
  return v[0];
}

template <int MODE, bool A_MN, bool FP16, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    xent_few_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const FewArgs a) {
  constexpr int T = NT / 2;  // tokens of one of the two warp groups
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t smem_base = smem_u32(smem_raw);
  if ((smem_base & 1023u) != 0) {  // the swizzled tiles need a 1024-byte aligned window: refuse to run otherwise
    overlapped_start();
    if (threadIdx.x == 0) atomicCAS(a.error_flag, 0, 5);
    return;
  }
  const uint32_t bars = smem_base + kFewOffBars;
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (kFewStages + s); };
  auto tfull_bar = [&](int b) { return bars + 8u * (2 * kFewStages + b); };
  auto tempty_bar = [&](int b) { return bars + 8u * (2 * kFewStages + 2 + b); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_raw + kFewOffBars + 8 * (2 * kFewStages + 4));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta_rank = cluster_rank();
  const int n_work = a.tiles * a.splits, first = blockIdx.x >> 1, step = gridDim.x >> 1;
  const int chunks = MODE == kOut ? 1 : a.chunks;
  auto split_begin = [&](int split) { return (int)((long long)split * a.k_blocks / a.splits); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kFewStages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull_bar(b), 1);
      mbar_init(tempty_bar(b), 2 * 8);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers exist before anything is sent to them
  fence_after_sync();
  const uint32_t tmem_base = *((volatile uint32_t*)tmem_slot);
  overlapped_start();  // nothing of global memory was touched so far
  if (MODE == kOut && a.tickets && blockIdx.x == 0 && (int)threadIdx.x < a.rows) a.tickets[threadIdx.x] = 0;

  if (warp == 0) {
    if (lane == 0) {  // TMA producer
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t leader_full0 = map_to_cta(full_bar(0), 0u);
      for (int work = first; work < n_work && ok; work += step) {
        const int split = work / a.tiles, m0 = (work - split * a.tiles) * 256 + (int)cta_rank * 128;
        for (int kb = split_begin(split); kb < split_begin(split + 1); ++kb) {
          if (!mbar_wait(empty_bar(s), ph ^ 1u, a.error_flag, 1)) {
            ok = false;
            break;
          }
          if (cta_rank == 0) mbar_expect_tx(full_bar(s), 2 * kOperandBytes + NT * 128);
          const uint32_t fb = leader_full0 + 8u * s, sa = smem_base + s * kFewStageBytes, sb = sa + kOperandBytes;
          const int k0 = kb * BK;
          if constexpr (A_MN) {
            tma_load_2d_pair(sa, &map_a, fb, m0, k0);
            tma_load_2d_pair(sa + kOperandBytes / 2, &map_a, fb, m0 + 64, k0);
          } else {
            tma_load_2d_pair(sa, &map_a, fb, k0, m0);
          }
          tma_load_2d_pair(sb, &map_b, fb, k0, (int)cta_rank * T);
          if (++s == kFewStages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // the leader's releases of this CTA's stages arrive asynchronously: see the last one of every stage land
      for (int q = 0; q < kFewStages && ok; ++q) {
        if (!mbar_wait(empty_bar(s), ph ^ 1u, a.error_flag, 1)) ok = false;
        if (++s == kFewStages) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (!ok) settle();
    }
  } else if (warp == 1) {
    if (lane == 0 && cta_rank == 0) {  // MMA issuer
      int s = 0, it = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int work = first; work < n_work && ok; work += step) {
        const int split = work / a.tiles, begin = split_begin(split), count = split_begin(split + 1) - begin;
        // floor(chunk count / chunks); with up to 2^16 chunks (2^26 features) no product here leaves 32 bits
        const unsigned each = (unsigned)count / (unsigned)chunks, more = (unsigned)count - each * (unsigned)chunks;
        auto chunk_begin = [&](unsigned chunk) { return (int)(chunk * each + chunk * more / (unsigned)chunks); };
        for (int chunk = 0; chunk < chunks && ok; ++chunk, ++it) {
          const int buf = it & 1;
          if (!mbar_wait(tempty_bar(buf), (uint32_t)((it >> 1) & 1) ^ 1u, a.error_flag, 2)) {
            ok = false;
            break;
          }
          fence_after_sync();
          const uint32_t d_tmem = tmem_base + (uint32_t)(buf * kFewSums * NT);
          const int kb0 = chunk_begin(chunk), kb1 = chunk_begin(chunk + 1);
          for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(full_bar(s), ph, a.error_flag, 3)) {
              ok = false;
              break;
            }
            fence_after_sync();
            const uint32_t sa = smem_base + s * kFewStageBytes, sb = sa + kOperandBytes;
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              umma_f16_pair(d_tmem + (uint32_t)(k * NT), A_MN ? umma_desc_mn(sa + k * 2048) : umma_desc(sa + k * 32), umma_desc(sb + k * 32),
                            a.idesc, kb > kb0 ? 1u : 0u);
            umma_commit_pair(empty_bar(s));
            if (++s == kFewStages) {
              s = 0;
              ph ^= 1u;
            }
          }
          if (ok) umma_commit_pair(tfull_bar(buf));
        }
      }
      if (!ok) settle();
    }
  } else {
    // epilogue: lanes are rows of the long operand, warps 2-5 and 6-9 take half of the tokens each
    const int quarter = warp & 3, half = (warp - 2) >> 2, token0 = half * T;
    const uint32_t leader_tempty0 = map_to_cta(tempty_bar(0), 0u);
    float* maxima = reinterpret_cast<float*>(smem_raw + kFewOffShared) + half * (4 * 32);
    float* sums = maxima + 2 * 4 * 32;
    const int live_tokens = max(0, min(T, a.rows - token0));
    long long label = -1;
    if constexpr (MODE != kOut)
      if (lane < live_tokens) label = __ldg(a.labels + token0 + lane);  // of the lane's token
    int it = 0;
    bool ok = true;  // after a wait that gave up a warp does no work, but meets the others at their barriers
    for (int work = first; work < n_work; work += step) {
      const int split = work / a.tiles;
      const long long base = (long long)(work - split * a.tiles) * 256 + cta_rank * 128 + quarter * 32, row = base + lane;
      const bool live = row < a.M;
      float bias = 0.f;
      if constexpr (MODE != kOut)
        if (a.bias && live) bias = __ldg(a.bias + row);
      float z[T];
      for (int chunk = 0; chunk < chunks && ok; ++chunk, ++it) {
        const int buf = it & 1;
        ok = mbar_wait(tfull_bar(buf), (uint32_t)((it >> 1) & 1), a.error_flag, 4);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after_sync();
        const uint32_t taddr = tmem_base + (uint32_t)(buf * kFewSums * NT + token0) + ((uint32_t)(quarter * 32) << 16);
#pragma unroll
        for (int k = 0; k < kFewSums; ++k) {
          uint32_t v[T];
#pragma unroll
          for (int j = 0; j < T; j += 16) tmem_ld16(taddr + k * NT + j, v + j);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < T; ++j) z[j] = chunk == 0 && k == 0 ? __uint_as_float(v[j]) : z[j] + __uint_as_float(v[j]);
        }
        fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(leader_tempty0 + 8u * buf);
      }
      if constexpr (MODE == kOut) {
        if (!ok) {  // NaN for what is left, as in xent_product_kernel
          if (live)
            for (int j = 0; j < live_tokens; ++j) {
              if (a.out32) a.out32[((long long)split * a.rows + token0 + j) * a.ld32 + row] = NAN;
              else a.out16[(long long)(token0 + j) * a.M + row] = 0x7fffu;
            }
          continue;
        }
        const float scale = a.scale ? __ldg(a.scale) : 1.0f;
        if (live) {
#pragma unroll
          for (int j = 0; j < T; ++j) {
            if (j >= live_tokens) break;
            if (a.out32) a.out32[((long long)split * a.rows + token0 + j) * a.ld32 + row] = z[j] * scale;
            else a.out16[(long long)(token0 + j) * a.M + row] = pack1<FP16>(z[j] * scale);
          }
        }
      } else {
        if (!ok) {
          asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
          asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
          continue;
        }
#pragma unroll
        for (int j = 0; j < T; ++j) z[j] = live ? z[j] + bias : -INFINITY;
        const long long at = label - base;  // lane of this warp that holds the lane's token's label
        if (__any_sync(0xffffffffu, at >= 0 && at < 32)) {
#pragma unroll
          for (int j = 0; j < T; ++j) {
            const long long where = __shfl_sync(0xffffffffu, at, j);
            if (j < live_tokens && where == lane && live) a.label_logit[token0 + j] = z[j];
          }
        }
        const float warp_max = reduce_lanes<T, true>(z, lane);
        if (lane < T) maxima[quarter * 32 + lane] = warp_max;
        asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
        float m = -INFINITY;  // of the lane's token (lane % T) over the slice
#pragma unroll
        for (int q = 0; q < 4; ++q) m = fmaxf(m, maxima[q * 32 + (lane & (T - 1))]);
#pragma unroll
        for (int j = 0; j < T; ++j) {
          const float top = __shfl_sync(0xffffffffu, m, j);
          z[j] = exp2_approx((z[j] - (top == -INFINITY ? 0.f : top)) * kLog2e);
        }
        const float warp_sum32 = reduce_lanes<T, false>(z, lane);
        if (lane < T) sums[quarter * 32 + lane] = warp_sum32;
        asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");
        if (quarter == 0 && lane < live_tokens && base < a.M) {
          const float s = (sums[lane] + sums[32 + lane]) + (sums[64 + lane] + sums[96 + lane]);
          a.stats[(base / kSlice) * a.ld_stats + token0 + lane] = make_float2(m, s);
        }
        if constexpr (MODE != kLoss) {
          if (live) {
#pragma unroll
            for (int j = 0; j < T; ++j) {
              if (j >= live_tokens) break;
              const unsigned short kept = pack1<FP16>(z[j] * kProbScale<FP16>);
              const long long to = (long long)(token0 + j) * a.ld_e + row;
              a.e[to] = kept;
              if constexpr (MODE == kProbLow) a.e_low[to] = pack1<FP16>(fmaf(z[j], kProbScale<FP16>, -unpack2<FP16>(kept).x));
            }
          }
        }
      }
    }
    if (!ok) settle();
  }
  fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the pair leaves together
  if (warp == 1) {
    fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
}

// What the rows count for, by one block (a fixed order, and the counts are whole numbers). `scalars`: [0]
// scale of the gradient (the rows' weights are stored as fractions of the largest one, so that any upstream gradient
// fits the 16-bit type), [1] the weights' inverse scale, [2] factor of the summed loss.
struct Weights {
  const long long* labels;  // of all rows
  long long rows;
  int reduction;
  const float* grad_loss;
  float prob_scale;
  float* scalars;           // null: not wanted
};
__device__ void row_weights(const Weights& a, long long ignore_index) {
  __shared__ unsigned long long count_part[32];
  __shared__ float max_part[32];
  unsigned long long count = 0;
  float top = 0.f;
#pragma unroll 4
  for (long long i = threadIdx.x; i < a.rows; i += blockDim.x) {
    const bool valid = a.labels[i] != ignore_index;
    count += valid;
    if (a.reduction == EVOX_REDUCE_NONE && a.grad_loss && valid) {
      const float g = fabsf(a.grad_loss[i]);
      if (g <= 3.0e38f) top = fmaxf(top, g);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    count += __shfl_xor_sync(0xffffffffu, count, o);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if ((threadIdx.x & 31) == 0) {
    count_part[threadIdx.x >> 5] = count;
    max_part[threadIdx.x >> 5] = top;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < (int)blockDim.x / 32; ++w) {
      count += count_part[w];
      top = fmaxf(top, max_part[w]);
    }
    const float per_row = a.reduction == EVOX_REDUCE_MEAN ? 1.0f / (float)count : 1.0f;  // no valid row: the mean is 0 / 0
    float scale;
    if (a.reduction == EVOX_REDUCE_NONE)
      scale = a.grad_loss ? (top > 1.0e-36f ? top : 1.0f) : 1.0f;
    else
      scale = count == 0 ? 0.f : per_row * (a.grad_loss ? a.grad_loss[0] : 1.0f);
    a.scalars[0] = scale / a.prob_scale;
    a.scalars[1] = 1.0f / scale;
    a.scalars[2] = per_row;
  }
}

// loss[i] and norm[i] = (maximum, 1 / sum of exponentials) from the slices' pairs: lanes are rows, warps share the slices.
// The two stay apart: added into one log-sum-exp, the logarithm would vanish next to a maximum of large size. A label outside the
// vocabulary that is not ignore_index gives NaN (and NaN gradients): loud, and nothing is read out of bounds. Where the status
// word says that a launch gave up every loss is NaN, and by way of norm every gradient: the slices may never have been written.
__global__ void __launch_bounds__(1024)
    xent_finish_kernel(const float2* __restrict__ stats, long long ld_stats, int slices, const float* __restrict__ label_logit,
                       const long long* __restrict__ labels, long long label_period, long long ignore_index, long long rows, long long vocab,
                       float2* __restrict__ norm, float* __restrict__ loss, const int* __restrict__ status, const Weights weights) {
  overlapped_start();
  if (weights.scalars && blockIdx.x == gridDim.x - 1) {  // one block more than the rows need
    row_weights(weights, ignore_index);
    return;
  }
  __shared__ float sm[32][33], ss[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = (long long)blockIdx.x * 32 + lane;
  const bool failed = __ldcg(status) != 0;
  float m = -INFINITY, s = 0.f;
  if (row < rows) {
#pragma unroll 4
    for (int j = warp; j < slices; j += 32) {
      const float2 p = __ldg(stats + (long long)j * ld_stats + row);
      const float top = fmaxf(m, p.x);
      s = s * rescale_to(m, top) + p.y * rescale_to(p.x, top);
      m = top;
    }
  }
  sm[warp][lane] = m;
  ss[warp][lane] = s;
  __syncthreads();
  // a warp per row: lanes are the 32 partial results
  const long long mine = (long long)blockIdx.x * 32 + warp;
  if (mine >= rows) return;
  const float pm = sm[lane][warp];
  m = pm;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  s = warp_sum(ss[lane][warp] * expf(pm - (m == -INFINITY ? 0.f : m)));
  if (lane == 0) {
    const long long y = labels[mine % label_period];
    const bool ignored = y == ignore_index, outside = !ignored && (y < 0 || y >= vocab);
    if (norm) norm[mine] = make_float2(m, outside || failed ? NAN : 1.0f / s);
    loss[mine] = failed ? NAN : ignored ? 0.f : (outside ? NAN : (m - label_logit[mine]) + logf(s));
  }
}

// Few rows whose logits came as partial sums over pieces of the hidden features (partial[split][row][ld]): 2,048 words of a
// row per block; the last block of a row joins the blocks' (maximum, sum) in their order. One more block of the last grid
// row computes the weights. A warp's first maximum may be of words past the vocabulary (-inf): rescale_to copes.
constexpr int kJoinWords = 2048;
__global__ void __launch_bounds__(256)
    xent_logits_kernel(const float* __restrict__ partial, int splits, long long ld, const float* __restrict__ bias,
                       const long long* __restrict__ labels, long long ignore_index, int rows, long long vocab, float2* parts,
                       float* label_logit, int* tickets, float* __restrict__ loss, const int* __restrict__ status, const Weights weights) {
  overlapped_start();
  const int row = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (row == rows) {
    if (blockIdx.x == 0) row_weights(weights, ignore_index);
    return;
  }
  __shared__ float sm[8], ss[8];
  __shared__ int last;
  const bool failed = __ldcg(status) != 0;
  const long long label = labels[row];
  float z[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // words 4 t .. 4 t + 3 of either half of the block's
    const long long v = (long long)blockIdx.x * kJoinWords + h * (kJoinWords / 2) + threadIdx.x * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (v < vocab) {  // lines hold a multiple of eight words
#pragma unroll 4
      for (int k = 0; k < splits; ++k) {
        const float4 p = __ldcs(reinterpret_cast<const float4*>(partial + ((long long)k * rows + row) * ld + v));
        sum.x += p.x; sum.y += p.y; sum.z += p.z; sum.w += p.w;
      }
    }
    const float got[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      z[4 * h + j] = v + j < vocab ? got[j] + (bias ? __ldg(bias + v + j) : 0.f) : -INFINITY;
      if (v + j == label && v + j < vocab) label_logit[row] = z[4 * h + j];
    }
  }
  float m = z[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) m = fmaxf(m, z[j]);
  m = fmaxf(m, -INFINITY);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) sm[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, sm[w]);
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) s += rescale_to(z[j], m);
  s = warp_sum(s);
  if (lane == 0) ss[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.f;
    for (int w = 0; w < 8; ++w) s += ss[w];
    parts[(long long)row * gridDim.x + blockIdx.x] = make_float2(m, s);
    __threadfence();  // also of the label's logit, which another thread stored before the barriers above
    last = atomicAdd(tickets + row, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last || warp != 0) return;
  __threadfence();
  m = -INFINITY;
  s = 0.f;
  for (int b = lane; b < (int)gridDim.x; b += 32) {
    const float2 p = __ldcg(parts + (long long)row * gridDim.x + b);
    const float top = fmaxf(m, p.x);
    s = s * rescale_to(m, top) + p.y * rescale_to(p.x, top);
    m = top;
  }
  const float mine = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  s = warp_sum(s * rescale_to(mine, m));
  if (lane == 0) {
    const bool ignored = label == ignore_index, outside = !ignored && (label < 0 || label >= vocab);
    loss[row] = failed ? NAN : ignored ? 0.f : (outside ? NAN : (m - __ldcg(label_logit + row)) + logf(s));
  }
}

// One block of 256 threads: out = scalars[2] * the sum of the losses, in 64 bits and a fixed order.
__device__ void sum_losses(const float* __restrict__ loss, long long rows, const float* __restrict__ scalars, float* __restrict__ out) {
  __shared__ double part[8];
  double s = 0.0;
#pragma unroll 8
  for (long long i = threadIdx.x; i < rows; i += 256) s += (double)loss[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) s += part[w];
    out[0] = (float)(s * (double)scalars[2]);
  }
}

constexpr int kRescaleColumns = 1024;  // columns of a block of the rescaling pass
// e -> g in place (see the head of the file), `block_rows` (at most 32) rows x 1,024 columns per block, eight columns per
// thread; column sums of the block's rows for the bias gradient, which is a 32-bit result: they take e with what its
// rounding left. The blocks of one more grid row copy the hidden states for the weight gradient, with zeros where the
// label is ignored: 0 x inf in a padded row must not reach dw. The first block of another one sums the losses of
// all rows once they are there.
template <bool FP16, bool BIAS>
__global__ void __launch_bounds__(256, BIAS ? 3 : 5)
    xent_rescale_kernel(unsigned short* __restrict__ e, const unsigned short* __restrict__ e_low, long long ld_e,
                        const float2* __restrict__ stats, long long ld_stats, int slices, const float2* __restrict__ norm,
                        const long long* __restrict__ labels, long long ignore_index, const float* __restrict__ grad_loss, int per_row,
                        const float* __restrict__ scalars, long long rows, int block_rows, long long vocab,
                        float* __restrict__ bias_partial, const unsigned short* __restrict__ h, long long ld_h, long long hidden,
                        unsigned short* __restrict__ h_out, long long ld_h_out, int column_blocks, const float* __restrict__ loss, long long all_rows,
                        float* __restrict__ loss_out) {
  overlapped_start();
  if ((int)blockIdx.y > column_blocks) {
    if (blockIdx.x == 0 && loss_out) sum_losses(loss, all_rows, scalars, loss_out);
    return;
  }
  const long long row0 = (long long)blockIdx.x * block_rows;
  const int n_rows = (int)min((long long)block_rows, rows - row0);
  const int tid = threadIdx.x;
  if ((int)blockIdx.y == column_blocks) {
    if (!h_out) return;
    const int pieces = (int)(ld_h_out / 8);
    for (int r = 0; r < n_rows; ++r) {
      const bool keep = labels[row0 + r] != ignore_index;
      const unsigned short* from = h + (row0 + r) * ld_h;
      unsigned short* to = h_out + (row0 + r) * ld_h_out;
      for (int i = tid; i < pieces; i += 256) {
        const int c = i * 8;
        uint4 p = make_uint4(0u, 0u, 0u, 0u);
        if (keep && c + 8 <= hidden) {
          p = __ldg(reinterpret_cast<const uint4*>(from + c));
        } else if (keep) {  // the row may end here
          unsigned short* q = reinterpret_cast<unsigned short*>(&p);
          for (int j = 0; j < 8; ++j)
            if (c + j < hidden) q[j] = from[c + j];
        }
        *reinterpret_cast<uint4*>(to + c) = p;
      }
    }
    return;
  }
  __shared__ float factor[32][8];
  __shared__ float weight[32];
  __shared__ int target[32];
  __shared__ float sums[128][8];
  // backwards: the columns that the product wrote last are still in the L2 cache, and those written here last are the first
  // that the next product reads
  const long long col_base = (long long)(column_blocks - 1 - (int)blockIdx.y) * kRescaleColumns;
  const int group = tid & 127, part = tid >> 7;  // eight columns; even or odd rows
  const long long col = col_base + group * 8;
  unsigned short* column = e + row0 * ld_e + col;
  // four rows at once; the first four are on their way while the factors are looked up
  uint4 p[4];
  auto fetch = [&](int r0) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r0 + 2 * i < n_rows) p[i] = *reinterpret_cast<const uint4*>(column + (r0 + 2 * i) * ld_e);
  };
  if (col < ld_e) fetch(part);
  {  // one (row, slice) per thread
    const int r = tid & 31, s = tid >> 5;
    const long long slice = col_base / kSlice + s;
    float f = 0.f, w = 0.f;
    int at = -1;
    if (r < n_rows) {
      const long long y = labels[row0 + r], d = y - col_base;
      if (y != ignore_index) {
        w = per_row && grad_loss ? grad_loss[row0 + r] * scalars[1] : 1.0f;
        if (d >= 0 && d < 1024) at = (int)d;
      }
      // w = 0 (an ignored row) stays 0 whatever the row holds: 0 x NaN is not formed
      if (w != 0.f && slice < slices) {
        const float2 q = norm[row0 + r];
        f = rescale_to(stats[slice * ld_stats + row0 + r].x, q.x) * q.y * w;
      }
    }
    factor[r][s] = f;
    if (s == 0) {
      weight[r] = w;
      target[r] = at;
    }
  }
  __syncthreads();
  float acc[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = 0.f;
  if (col < ld_e) {
    auto one = [&](int r, uint4 p) {
      const float f = factor[r][group >> 4], w = weight[r];
      uint32_t* word = reinterpret_cast<uint32_t*>(&p);
      uint4 low = make_uint4(0u, 0u, 0u, 0u);
      if (BIAS && w != 0.f) low = __ldcs(reinterpret_cast<const uint4*>(e_low + (row0 + r) * ld_e + col));
      const uint32_t lw[4] = {low.x, low.y, low.z, low.w};
      const int t = target[r] - group * 8;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float2 x = unpack2<FP16>(word[j]);
        const float2 y = unpack2<FP16>(lw[j]);
        const float h0 = t == 2 * j ? kProbScale<FP16> * w : 0.f, h1 = t == 2 * j + 1 ? kProbScale<FP16> * w : 0.f;
        if (BIAS && w != 0.f) {
          acc[2 * j] += (x.x + y.x) * f - h0;
          acc[2 * j + 1] += (x.y + y.y) * f - h1;
        }
        word[j] = pack2<FP16>(fmaf(x.x, f, -h0), fmaf(x.y, f, -h1));
      }
      return w != 0.f ? p : make_uint4(0u, 0u, 0u, 0u);
    };
    for (int r0 = part; r0 < n_rows; r0 += 8) {
      if (r0 != part) fetch(r0);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (r0 + 2 * i < n_rows) *reinterpret_cast<uint4*>(column + (r0 + 2 * i) * ld_e) = one(r0 + 2 * i, p[i]);
    }
  }
  if constexpr (BIAS) {
    if (part == 1) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sums[group][j] = acc[j];
    }
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < vocab) bias_partial[(long long)blockIdx.x * vocab + col + j] = acc[j] + sums[group][j];
    }
  }
}

// The end of a gradient: up to two products whose reduction was divided (sum over the splits, in their order, of partial
// results that are scaled already) and the bias gradient (scale times the sum over the row blocks, in their order; added to
// what the earlier row chunks left). Blocks are dealt to the three in turn.
struct Join {
  const float* partial;  // [splits][rows][ld32]
  unsigned short* out;   // [rows][cols], 16 bits
  long long rows, cols, ld32;
  int splits, blocks;    // blocks: 0 if there is nothing to join
};
struct BiasSum {
  const float* partial;  // [row_blocks][vocab]
  float* out;
  const float* scale;
  long long vocab;
  int row_blocks, add, blocks;
};
template <bool FP16>
__global__ void __launch_bounds__(256) xent_join_kernel(const Join dh, const Join dw, const BiasSum db) {
  overlapped_start();
  int block = blockIdx.x;
  if (block < db.blocks) {
    // 32 columns, the row blocks dealt to eight warps
    __shared__ float part[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long v = (long long)block * 32 + lane;
    float s = 0.f;
    if (v < db.vocab) {
#pragma unroll 8
      for (int b = warp; b < db.row_blocks; b += 8) s += __ldg(db.partial + (long long)b * db.vocab + v);
    }
    part[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && v < db.vocab) {
      for (int w = 1; w < 8; ++w) s += part[w][lane];
      s *= db.scale[0];
      db.out[v] = db.add ? db.out[v] + s : s;
    }
    return;
  }
  block -= db.blocks;
  const Join a = block < dh.blocks ? dh : dw;
  if (block >= dh.blocks) block -= dh.blocks;
  const long long quads = (a.cols + 3) / 4, n = a.rows * quads;
  for (long long i = (long long)block * 256 + threadIdx.x; i < n; i += (long long)a.blocks * 256) {
    const long long r = i / quads, c = (i - r * quads) * 4;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < a.splits; ++k) {
      const float4 p = __ldcs(reinterpret_cast<const float4*>(a.partial + ((long long)k * a.rows + r) * a.ld32 + c));
      s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
    }
    unsigned short* to = a.out + r * a.cols + c;
    if (a.cols % 4 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 7u) == 0) {
      *reinterpret_cast<uint2*>(to) = make_uint2(pack2<FP16>(s.x, s.y), pack2<FP16>(s.z, s.w));
    } else {
      const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < a.cols) to[j] = pack1<FP16>(v[j]);
    }
  }
}

// Sum of the rows' losses times the reduction's factor: one block, 64-bit sums in a fixed order.
__global__ void __launch_bounds__(256) xent_loss_sum_kernel(const float* __restrict__ loss, long long rows, const float* __restrict__ scalars, float* __restrict__ out) {
  overlapped_start();
  sum_losses(loss, rows, scalars, out);
}

// Operands whose rows do not start on 16-byte boundaries (a hidden size or a stride that is no multiple of 8, an odd start)
// are copied to rows that do, which is what TMA reads: one launch for both, eight columns per thread.
struct Align {
  const unsigned short* from;  // null: this operand is used as it is
  unsigned short* to;
  long long rows, ld_from, ld_to, cols;
};
__global__ void __launch_bounds__(256) xent_align_kernel(const Align h, const Align w) {
  overlapped_start();
  const long long n_h = h.from ? h.rows * (h.ld_to / 8) : 0, n_w = w.from ? w.rows * (w.ld_to / 8) : 0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n_h + n_w; i += (long long)gridDim.x * 256) {
    const bool first = i < n_h;
    const Align& a = first ? h : w;
    const long long q = first ? i : i - n_h, r = q / (a.ld_to / 8), c = (q - r * (a.ld_to / 8)) * 8;
    const unsigned short* src = a.from + r * a.ld_from + c;
    uint4 p = make_uint4(0u, 0u, 0u, 0u);
    if (c + 8 <= a.cols && (reinterpret_cast<uintptr_t>(src) & 3u) == 0) {
      const uint32_t* s32 = reinterpret_cast<const uint32_t*>(src);
      p = make_uint4(__ldg(s32), __ldg(s32 + 1), __ldg(s32 + 2), __ldg(s32 + 3));
    } else {
      unsigned short* e = reinterpret_cast<unsigned short*>(&p);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < a.cols) e[j] = __ldg(src + j);
    }
    *reinterpret_cast<uint4*>(a.to + r * a.ld_to + c) = p;
  }
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
long long up(long long x, long long m) { return (x + m - 1) / m * m; }

// Map of a 16-bit matrix (`outer` lines of `inner` elements, `ld` apart) with boxes of 64 elements x `box_outer` lines.
int map_16(CUtensorMap* map, const void* base, long long inner, long long outer, long long ld, int box_outer, bool fp16) {
  EncodeTiledFn fn;
  if (int rc = encode_fn(&fn)) return rc;
  const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {64u, (cuuint32_t)box_outer};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims,
                        strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  EVOX_REQUIRE(r == CUDA_SUCCESS, EVOX_ERR_CUDA, "linear_cross_entropy: cuTensorMapEncodeTiled failed with code %d", (int)r);
  return EVOX_OK;
}

// Lets a kernel use that much shared memory, once per device (bits of `allowed`; devices beyond the 64th every time).
template <typename K>
int allow_shared_memory(K kernel, uint32_t bytes, std::atomic<unsigned long long>& allowed) {
  int dev = 0;
  EVOX_CUDA(cudaGetDevice(&dev));
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0ull;
  if (allowed.load(std::memory_order_relaxed) & bit) return EVOX_OK;
  EVOX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return EVOX_OK;
}

// fp32 accumulator, both operands of the one 16-bit type, 256 x 256; operands contiguous along their rows at bits 15 and 16.
template <bool FP16>
void describe(Product& p, bool a_mn, bool b_mn) {
  p.tiles_m = (int)((p.M + TM - 1) / TM);
  p.tiles_n = (int)((p.N + TN - 1) / TN);
  const int fast = p.m_fast ? p.tiles_m : p.tiles_n;
  if (p.group > fast) p.group = fast;
  p.a_mn = a_mn;
  p.idesc = (1u << 4) | ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(TM >> 4) << 24) | (FP16 ? 0u : (1u << 7) | (1u << 10)) |
            (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
}

// Cost of a work item in blocks of the reduction; below nine blocks the epilogue is what takes the time.
long long item_cost(const Product& p) {
  const long long kb = (p.k_blocks + p.splits - 1) / p.splits;
  return kb < 9 ? 9 : kb;
}

// How the work items are dealt; returns the longest pair's cost.
long long deal(ProductArgs& a) {
  for (int i = 0; i < 2; ++i) a.items[i] = a.p[i].M > 0 ? a.p[i].tiles_m * a.p[i].tiles_n * a.p[i].splits : 0;
  const long long slots = sm_count() / 2, items0 = a.items[0], items1 = a.items[1];
  const long long c0 = items0 > 0 ? item_cost(a.p[0]) : 0, c1 = items1 > 0 ? item_cost(a.p[1]) : 0;
  a.pairs = (int)(items0 + items1 < slots ? items0 + items1 : slots);
  a.heavy = (int)(items0 % a.pairs);
  a.per_heavy = a.early = 0;
  const long long light = items0 / a.pairs * c0, heavy = light + c0, fair = (items0 * c0 + items1 * c1) / a.pairs;
  if (items1 == 0) return a.heavy ? heavy : light;
  long long best = -1;
  for (long long per = fair > heavy ? (fair - heavy) / c1 : 0, last = per + 1; per <= last; ++per) {  // whole items: up or down
    const long long left = items1 - per * a.pairs, others = a.pairs - a.heavy;
    const long long early = left > 0 ? (left + others - 1) / others : 0;
    const long long with = a.heavy ? heavy + per * c1 : 0, without = light + (early + per) * c1, end = with > without ? with : without;
    if (best < 0 || end < best) {
      best = end;
      a.per_heavy = (int)per;
      a.early = (int)early;
    }
  }
  return best;
}

template <int MODE, bool FP16>
int launch_product(const Maps& maps, ProductArgs& a, cudaStream_t stream) {
  if (a.stage_bytes == 0) a.stage_bytes = 2 * kStageBytes;
  if (MODE == kOut && a.p[0].M > 0 && a.p[1].M > 0) {
    // Together neither product waits for the other's last tiles, but they compete for the L2 cache: they share a launch where
    // that saves 3 % of the longest pair's work. Whole gradient steps, together and apart: 500 x 1,024 x 8,000 42 and 51 us,
    // 1,003 x 1,000 x 50,021 308 and 324, 2,048 x 2,048 x 32,768 605 and 614; 8,192 x 4,096 x 131,072, where
    // there is nothing to save, 23.5 and 22.1 ms.
    ProductArgs first = a, second = a;
    first.p[1].M = second.p[0].M = 0;
    const long long apart = deal(first) + deal(second), together = deal(a);
    if (apart * 100 < together * 103) {
      if (int rc = launch_product<MODE, FP16>(maps, first, stream)) return rc;
      return launch_product<MODE, FP16>(maps, second, stream);
    }
  } else {
    deal(a);
  }
  static std::atomic<unsigned long long> allowed{0};
  if (int rc = allow_shared_memory(xent_product_kernel<MODE, FP16>, kSmemBytes, allowed)) return rc;
  EVOX_CUDA(launch_overlapped(xent_product_kernel<MODE, FP16>, dim3((unsigned)(2 * a.pairs)), kThreads, kSmemBytes, 2, stream, maps, a));
  return EVOX_OK;
}

// Rows (or columns) of tiles that run together so that their operand, `bytes_per_tile` each, stays in the L2 cache
// next to what streams past it.
int resident_group(long long bytes_per_tile) {
  const long long g = (48ll << 20) / (bytes_per_tile > 0 ? bytes_per_tile : 1);
  return (int)(g < 1 ? 1 : (g > 1024 ? 1024 : g));
}

// Into how many work items per tile the reductions of dh (rows x hidden over vocab) and dw (vocab x hidden over rows) are
// divided: an item should not take longer than a pair's fair share of both, nor be shorter than eight blocks.
void gradient_splits(long long rows, long long hidden, long long vocab, int& dh, int& dw) {
  auto tiles = [](long long m, long long n) { return ((m + TM - 1) / TM) * ((n + TN - 1) / TN); };
  const long long kb_dh = (vocab + BK - 1) / BK, kb_dw = (rows + BK - 1) / BK;
  long long fair = (tiles(rows, hidden) * kb_dh + tiles(vocab, hidden) * kb_dw) / (sm_count() / 2);
  if (fair < 1) fair = 1;
  auto splits = [&](long long kb) {
    long long s = (kb + fair - 1) / fair;
    if (s > kb / 8) s = kb / 8;
    if (s > 16) s = 16;
    return (int)(s < 1 ? 1 : s);
  };
  dh = splits(kb_dh);
  dw = splits(kb_dw);
}

// Rows per block of the rescaling pass: 32, or 8 where that would leave half of the machine without blocks.
int rescale_rows(long long rows, long long vocab) {
  return ((rows + 31) / 32) * ((vocab + 1023) / 1024) >= 4ll * sm_count() ? 32 : 8;
}

// Work items per tile of a product with few tokens: one item per CTA pair (four were slower: 183 against 174 us for a gradient
// at 8 x 4,096 x 32,000), at least eight blocks of the reduction each.
int few_splits(long long M, long long K) {
  const long long tiles = (M + 255) / 256, pairs = sm_count() / 2, kb = (K + BK - 1) / BK;
  long long s = pairs / tiles;
  if (s > kb / 8) s = kb / 8;
  return (int)(s < 1 ? 1 : s);
}

// Into how many pieces the hidden features are divided for the loss of few rows, so that the weight's tiles (256 words and
// all features) become work items that the CTA pairs share evenly: the fewest waves of items, at 0.3 us per block of the
// reduction, against writing and reading the partial logits at about 4 TB/s (L2 cache).
int few_loss_splits(long long rows, long long hidden, long long vocab) {
  const long long tiles = (vocab + 255) / 256, pairs = sm_count() / 2, kb = (hidden + BK - 1) / BK;
  double best = 0.0;
  int splits = 1;
  for (int s = 1; s <= 16 && (s == 1 || kb / s >= 4); s *= 2) {
    const double product = 0.3 * (double)((tiles * s + pairs - 1) / pairs) * (double)((kb + s - 1) / s);
    const double cost = product + (s > 1 ? 1.0 + (double)(rows * vocab * s) * 8.0 / 4.0e6 : 0.0);
    if (s == 1 || cost < best) {
      best = cost;
      splits = s;
    }
  }
  return splits;
}

template <int MODE, bool A_MN, bool FP16, int NT>
int launch_few_nt(const CUtensorMap& map_a, const CUtensorMap& map_b, FewArgs& a, cudaStream_t stream) {
  a.tiles = (int)((a.M + 255) / 256);
  a.idesc = (1u << 4) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(256 >> 4) << 24) | (FP16 ? 0u : (1u << 7) | (1u << 10)) | (A_MN ? 1u << 15 : 0u);
  const long long n_work = (long long)a.tiles * a.splits, slots = sm_count() / 2, pairs = n_work < slots ? n_work : slots;
  static std::atomic<unsigned long long> allowed{0};
  if (int rc = allow_shared_memory(xent_few_kernel<MODE, A_MN, FP16, NT>, kFewSmemBytes, allowed)) return rc;
  EVOX_CUDA(launch_overlapped(xent_few_kernel<MODE, A_MN, FP16, NT>, dim3((unsigned)(2 * pairs)), kThreads, kFewSmemBytes, 2, stream, map_a, map_b, a));
  return EVOX_OK;
}

// The long operand through `map_a`, `a.rows` tokens (K-major lines of `line` elements, `ld` apart).
template <int MODE, bool A_MN, bool FP16>
int launch_few(const CUtensorMap& map_a, const void* tokens, long long line, long long ld, FewArgs& a, cudaStream_t stream) {
  CUtensorMap map_b;
  const bool small = a.rows <= 32;
  if (int rc = map_16(&map_b, tokens, line, a.rows, ld, small ? 16 : 32, FP16)) return rc;
  return small ? launch_few_nt<MODE, A_MN, FP16, 32>(map_a, map_b, a, stream) : launch_few_nt<MODE, A_MN, FP16, 64>(map_a, map_b, a, stream);
}

struct Carve {  // 256-byte aligned pieces of the workspace
  uint8_t* base;
  size_t used;
  template <class T>
  T* take(size_t count) {
    T* p = reinterpret_cast<T*>(base + used);
    used += (count * sizeof(T) + 255) / 256 * 256;
    return p;
  }
};

struct Buffers {
  unsigned short* h_aligned;
  unsigned short* w_aligned;
  float* scalars;
  float2* stats;
  float* label_logit;
  float2* norm;
  float* loss;
  unsigned short* e;
  unsigned short* e_low;  // with a bias gradient: it sums e itself, in 32 bits
  unsigned short* h_copy;
  float* bias_partial;
  float* partial_dh;  // products whose reduction is divided
  float* partial_dw;
  float* few_logits;  // partial logits of few rows, divided features
  float2* few_parts;
  int* few_tickets;
  float* dw_sum;      // running dw over the row chunks
};

// copies: bit 0: the hidden states are copied to aligned rows, bit 1: the weight is.
size_t layout(Buffers& b, void* base, long long rows, long long hidden, long long vocab, int copies, long long chunk, bool grad,
              bool with_bias) {
  Carve c{reinterpret_cast<uint8_t*>(base), 0};
  b.h_aligned = copies & 1 ? c.take<unsigned short>((size_t)rows * up(hidden, 8)) : nullptr;
  b.w_aligned = copies & 2 ? c.take<unsigned short>((size_t)vocab * up(hidden, 8)) : nullptr;
  const long long slices = (vocab + kSlice - 1) / kSlice;
  b.scalars = c.take<float>(4);
  b.stats = c.take<float2>((size_t)slices * chunk);
  b.label_logit = c.take<float>(chunk);
  b.loss = c.take<float>(rows);
  if (!grad && rows <= kFewRows) {
    const int splits = few_loss_splits(rows, hidden, vocab);
    b.few_logits = splits > 1 ? c.take<float>((size_t)splits * rows * up(vocab, 8)) : nullptr;
    b.few_parts = splits > 1 ? c.take<float2>((size_t)rows * ((vocab + kJoinWords - 1) / kJoinWords)) : nullptr;
    b.few_tickets = splits > 1 ? c.take<int>(rows) : nullptr;
  }
  if (grad) {
    b.norm = c.take<float2>(chunk);
    b.e = c.take<unsigned short>((size_t)chunk * up(vocab, 64));
    b.e_low = with_bias ? c.take<unsigned short>((size_t)chunk * up(vocab, 64)) : nullptr;
    b.h_copy = c.take<unsigned short>((size_t)chunk * up(hidden, 8));
    size_t sums = 0;  // of either chunk length
    for (long long r : {chunk, rows % chunk ? rows % chunk : chunk}) {
      const size_t n = (size_t)((r + rescale_rows(r, vocab) - 1) / rescale_rows(r, vocab));
      if (n > sums) sums = n;
    }
    b.bias_partial = with_bias ? c.take<float>(sums * vocab) : nullptr;
    size_t part_dh = 0;
    int splits_dw = 1;
    for (long long r : {chunk, rows % chunk ? rows % chunk : chunk}) {
      int splits;
      gradient_splits(r, hidden, vocab, splits, splits_dw);
      if (r <= kFewRows) splits = few_splits(hidden, vocab);
      if (splits > 1 && part_dh < (size_t)splits * r * up(hidden, 8)) part_dh = (size_t)splits * r * up(hidden, 8);
    }
    if (chunk < rows) splits_dw = 1;  // a running sum instead
    b.partial_dh = part_dh ? c.take<float>(part_dh) : nullptr;
    b.partial_dw = splits_dw > 1 ? c.take<float>((size_t)splits_dw * vocab * up(hidden, 8)) : nullptr;
    b.dw_sum = chunk < rows ? c.take<float>((size_t)vocab * up(hidden, 8)) : nullptr;
  }
  return c.used;
}

int check_operands(const char* what, const void* h, int64_t ld_h, const void* w, int64_t ld_w, int32_t dtype, const int64_t* labels,
                   int64_t rows, int64_t hidden, int64_t vocab, int32_t reduction, const float* loss, const void* workspace,
                   const int32_t* error_flag) {
  EVOX_REQUIRE(h && w && labels && loss && workspace && error_flag, EVOX_ERR_INVALID, "%s: NULL pointer", what);
  EVOX_REQUIRE(rows > 0 && hidden > 0 && vocab > 0 && rows < (1ll << 30) && hidden < (1ll << 26) && vocab < (1ll << 26), EVOX_ERR_INVALID,
               "%s: rows must be in [1, 2^30), hidden and vocab in [1, 2^26), got %lld, %lld, %lld", what, (long long)rows, (long long)hidden, (long long)vocab);
  EVOX_REQUIRE((rows + 255) / 256 * ((vocab + 255) / 256) < (1ll << 28) && (vocab + 255) / 256 * ((hidden + 255) / 256) < (1ll << 26),
               EVOX_ERR_INVALID, "%s: rows x vocab or vocab x hidden is too large", what);
  EVOX_REQUIRE(dtype == EVOX_DTYPE_BF16 || dtype == EVOX_DTYPE_FP16, EVOX_ERR_INVALID, "%s: operands must be bf16 or fp16", what);
  EVOX_REQUIRE(reduction == EVOX_REDUCE_NONE || reduction == EVOX_REDUCE_SUM || reduction == EVOX_REDUCE_MEAN, EVOX_ERR_INVALID,
               "%s: unknown reduction %d", what, reduction);
  EVOX_REQUIRE(ld_h >= hidden && ld_w >= hidden, EVOX_ERR_INVALID, "%s: row strides must be at least hidden", what);
  EVOX_REQUIRE(((uintptr_t)h & 1u) == 0 && ((uintptr_t)w & 1u) == 0, EVOX_ERR_INVALID, "%s: operands must be aligned to their elements", what);
  EVOX_REQUIRE(((uintptr_t)workspace & 255u) == 0, EVOX_ERR_INVALID, "%s: workspace must be 256-byte aligned", what);
  return EVOX_OK;
}

int copies_of(const void* h, long long ld_h, const void* w, long long ld_w) {
  return (aligned16(h) && ld_h % 8 == 0 ? 0 : 1) | (aligned16(w) && ld_w % 8 == 0 ? 0 : 2);
}

struct Head {
  const void* h;
  long long ld_h;
  const void* w;
  long long ld_w;
  const float* bias;
  const long long* labels;
  long long ignore_index, rows, hidden, vocab;
  int* error_flag;
  cudaStream_t stream;
};

int finish(const float2* stats, long long ld_stats, const float* label_logit, const long long* labels, long long label_period,
           long long ignore_index, long long rows, long long vocab, float2* norm, float* loss, const int* status, const Weights& weights,
           cudaStream_t stream) {
  const int slices = (int)((vocab + kSlice - 1) / kSlice);
  EVOX_CUDA(launch_overlapped(xent_finish_kernel, dim3((unsigned)((rows + 31) / 32 + (weights.scalars ? 1 : 0))), 1024, 0, 1, stream, stats,
                              ld_stats, slices, label_logit, labels, label_period, ignore_index, rows, vocab, norm, loss, status, weights));
  return EVOX_OK;
}

// Replaces operands that TMA cannot read by aligned copies in the workspace.
int align_operands(Head& x, const Buffers& b) {
  if (!b.h_aligned && !b.w_aligned) return EVOX_OK;
  const long long ld = up(x.hidden, 8);
  const Align h = {b.h_aligned ? (const unsigned short*)x.h : nullptr, b.h_aligned, x.rows, x.ld_h, ld, x.hidden};
  const Align w = {b.w_aligned ? (const unsigned short*)x.w : nullptr, b.w_aligned, x.vocab, x.ld_w, ld, x.hidden};
  const long long n = ((h.from ? x.rows : 0) + (w.from ? x.vocab : 0)) * (ld / 8), blocks = (n + 255) / 256, cap = 32ll * sm_count();
  EVOX_CUDA(launch_overlapped(xent_align_kernel, dim3((unsigned)(blocks < cap ? blocks : cap)), 256, 0, 1, x.stream, h, w));
  if (b.h_aligned) {
    x.h = b.h_aligned;
    x.ld_h = ld;
  }
  if (b.w_aligned) {
    x.w = b.w_aligned;
    x.ld_w = ld;
  }
  return EVOX_OK;
}

// Logits of `n` rows from `r0` on: (maximum, sum) per slice, the labels' logits, and the exponentials, as MODE says.
template <int MODE, bool FP16>
int logits_pass(const Head& x, const Buffers& b, long long r0, long long n, long long ld_stats) {
  const unsigned short* h = reinterpret_cast<const unsigned short*>(x.h) + r0 * x.ld_h;
  if (n <= kFewRows) {
    CUtensorMap map_a;
    if (int rc = map_16(&map_a, x.w, x.hidden, x.vocab, x.ld_w, 128, FP16)) return rc;
    FewArgs a = {};
    a.M = x.vocab;
    a.rows = (int)n;
    a.k_blocks = (int)((x.hidden + BK - 1) / BK);
    a.splits = 1;
    a.chunks = (a.k_blocks + kFewChunkBlocks - 1) / kFewChunkBlocks;
    a.error_flag = x.error_flag;
    a.bias = x.bias;
    a.labels = x.labels + r0;
    a.stats = b.stats;
    a.ld_stats = ld_stats;
    a.label_logit = b.label_logit;
    a.e = b.e;
    a.e_low = b.e_low;
    a.ld_e = up(x.vocab, 64);
    return launch_few<MODE, false, FP16>(map_a, h, x.hidden, x.ld_h, a, x.stream);
  }
  // up to 128 rows: copies of those rows only (whole groups of eight, the swizzle's unit), none in the second CTA. Rows of a
  // tile that nothing was copied to multiply whatever is there; their products are not used.
  const int box = n <= 128 ? (int)up(n, 8) : 128;
  Maps maps;
  if (int rc = map_16(&maps.a[0], h, x.hidden, n, x.ld_h, box, FP16)) return rc;
  if (int rc = map_16(&maps.b[0], x.w, x.hidden, x.vocab, x.ld_w, 128, FP16)) return rc;
  ProductArgs a = {};
  a.stage_bytes = n <= 128 ? 2 * kOperandBytes + (uint32_t)box * 128 : 2 * kStageBytes;
  Product& p = a.p[0];
  p.M = n;
  p.N = x.vocab;
  p.k_blocks = (int)((x.hidden + BK - 1) / BK);
  p.splits = 1;
  // a tensor-core accumulator truncates when it adds, a bias that grows with the number of additions: 1,024 hidden features
  // per accumulator, joined with rounding (mean loss at 16,384 x 4,096 x 131,072: 5.4e-7 off, 2.3e-6 with one accumulator)
  a.chunks = (p.k_blocks + kChunkBlocks - 1) / kChunkBlocks;
  p.m_fast = 1;  // the weight streams past, the hidden states stay in L2
  p.group = resident_group(2ll * TM * x.hidden);
  describe<FP16>(p, false, false);
  a.error_flag = x.error_flag;
  a.bias = x.bias;
  a.labels = x.labels + r0;
  a.stats = b.stats;
  a.ld_stats = ld_stats;
  a.label_logit = b.label_logit;
  maps.out[0] = maps.out[1] = maps.a[1] = maps.b[1] = maps.a[0];  // what this mode does not use
  if (MODE != kLoss) {
    const long long ld_e = up(x.vocab, 64);
    if (int rc = map_16(&maps.out[0], b.e, x.vocab, n, ld_e, 32, FP16)) return rc;
    if (MODE == kProbLow)
      if (int rc = map_16(&maps.out[1], b.e_low, x.vocab, n, ld_e, 32, FP16)) return rc;
  }
  return launch_product<MODE, FP16>(maps, a, x.stream);
}

// Losses of few rows with the features divided (few_loss_splits).
template <bool FP16>
int few_loss_pass(const Head& x, const Buffers& b, float* loss, const Weights& weights) {
  CUtensorMap map_a;
  if (int rc = map_16(&map_a, x.w, x.hidden, x.vocab, x.ld_w, 128, FP16)) return rc;
  FewArgs a = {};
  a.M = x.vocab;
  a.rows = (int)x.rows;
  a.k_blocks = (int)((x.hidden + BK - 1) / BK);
  a.splits = few_loss_splits(x.rows, x.hidden, x.vocab);
  a.error_flag = x.error_flag;
  a.out32 = b.few_logits;
  a.ld32 = up(x.vocab, 8);
  a.tickets = b.few_tickets;
  if (int rc = launch_few<kOut, false, FP16>(map_a, x.h, x.hidden, x.ld_h, a, x.stream)) return rc;
  const dim3 grid((unsigned)((x.vocab + kJoinWords - 1) / kJoinWords), (unsigned)(x.rows + (weights.scalars ? 1 : 0)));
  EVOX_CUDA(launch_overlapped(xent_logits_kernel, grid, 256, 0, 1, x.stream, b.few_logits, a.splits, a.ld32, x.bias, x.labels, x.ignore_index,
                              a.rows, x.vocab, b.few_parts, b.label_logit, b.few_tickets, loss, x.error_flag, weights));
  return EVOX_OK;
}

// Where product `i` of `a` goes: out (M x N, 16 bits, dense), through partial sums that `join` will add up where the reduction
// is divided, or by way of the running 32-bit sum over row chunks (`sum`; `first`, `last`: which chunk).
template <bool FP16>
int gradient_output(Maps& maps, ProductArgs& a, int i, void* out, float* partial, float* sum, bool first, bool last, Join* join) {
  Product& p = a.p[i];
  p.ld32 = up(p.N, 8);
  if (sum) {
    p.splits = 1;
    p.out32 = sum;
    p.add32 = !first;
    p.out16 = last ? out : nullptr;
  } else if (p.splits > 1) {
    p.out32 = partial;
    const long long blocks = (p.M * ((p.N + 3) / 4) + 255) / 256, cap = 16ll * sm_count();
    *join = Join{partial, reinterpret_cast<unsigned short*>(out), p.M, p.N, p.ld32, p.splits, (int)(blocks < cap ? blocks : cap)};
  } else {
    p.out16 = out;
  }
  p.tiled_out = p.out16 && p.N % 8 == 0 && aligned16(out);
  if (p.tiled_out) return map_16(&maps.out[i], out, p.N, p.M, p.N, 32, FP16);
  return EVOX_OK;
}

template <bool FP16>
int gradient_pass(const Head& x, const Buffers& b, long long chunk, int reduction, const float* grad_loss, float* loss, void* dh, void* dw,
                  float* db) {
  const int slices = (int)((x.vocab + kSlice - 1) / kSlice);
  const long long ld_e = up(x.vocab, 64), ld_copy = up(x.hidden, 8);
  const bool per_row = reduction == EVOX_REDUCE_NONE;
  float* row_loss = per_row ? loss : b.loss;
  for (long long r0 = 0; r0 < x.rows; r0 += chunk) {
    const long long n = x.rows - r0 < chunk ? x.rows - r0 : chunk;
    const bool first = r0 == 0, last = r0 + n == x.rows;
    if (int rc = b.e_low ? logits_pass<kProbLow, FP16>(x, b, r0, n, chunk) : logits_pass<kProb, FP16>(x, b, r0, n, chunk)) return rc;
    const Weights weights = {x.labels, x.rows, reduction, grad_loss, kProbScale<FP16>, first ? b.scalars : nullptr};
    if (int rc = finish(b.stats, chunk, b.label_logit, x.labels + r0, n, x.ignore_index, n, x.vocab, b.norm, row_loss + r0, x.error_flag, weights,
                        x.stream))
      return rc;
    const unsigned short* h = reinterpret_cast<const unsigned short*>(x.h) + r0 * x.ld_h;
    const int column_blocks = (int)((x.vocab + kRescaleColumns - 1) / kRescaleColumns), block_rows = rescale_rows(n, x.vocab);
    const int row_blocks = (int)((n + block_rows - 1) / block_rows);
    const bool sum_here = last && !per_row;
    EVOX_CUDA(launch_overlapped(
        db ? xent_rescale_kernel<FP16, true> : xent_rescale_kernel<FP16, false>, dim3((unsigned)row_blocks, (unsigned)(column_blocks + (sum_here ? 2 : dw ? 1 : 0))), 256, 0, 1, x.stream, b.e, b.e_low, ld_e, b.stats, chunk, slices, b.norm, x.labels + r0, x.ignore_index, grad_loss && per_row ? grad_loss + r0 : nullptr,
        per_row, b.scalars, n, block_rows, x.vocab, db ? b.bias_partial : nullptr, h, x.ld_h, x.hidden, dw ? b.h_copy : nullptr, ld_copy,
        column_blocks, row_loss, x.rows, sum_here ? loss : nullptr));
    Join join_dh = {}, join_dw = {};
    unsigned short* dh_rows = dh ? reinterpret_cast<unsigned short*>(dh) + r0 * x.hidden : nullptr;
    const bool few = n <= kFewRows;
    if (dh && few) {
      CUtensorMap map_a;
      if (int rc = map_16(&map_a, x.w, x.hidden, x.vocab, x.ld_w, 64, FP16)) return rc;
      FewArgs a = {};
      a.M = x.hidden;
      a.rows = (int)n;
      a.k_blocks = (int)((x.vocab + BK - 1) / BK);
      a.splits = few_splits(x.hidden, x.vocab);
      a.error_flag = x.error_flag;
      a.scale = b.scalars;
      a.ld32 = up(x.hidden, 8);
      if (a.splits > 1) a.out32 = b.partial_dh;
      else a.out16 = dh_rows;
      if (int rc = launch_few<kOut, true, FP16>(map_a, b.e, x.vocab, ld_e, a, x.stream)) return rc;
      if (a.splits > 1) {
        const long long blocks = (n * ((x.hidden + 3) / 4) + 255) / 256, cap = 16ll * sm_count();
        join_dh = Join{b.partial_dh, dh_rows, n, x.hidden, a.ld32, a.splits, (int)(blocks < cap ? blocks : cap)};
      }
    }
    if ((dh && !few) || dw) {
      Maps maps;
      ProductArgs a = {};
      a.error_flag = x.error_flag;
      a.scale = b.scalars;
      gradient_splits(n, x.hidden, x.vocab, a.p[0].splits, a.p[1].splits);
      if (int rc = map_16(&maps.a[0], b.e, x.vocab, n, ld_e, 128, FP16)) return rc;
      maps.a[1] = maps.b[0] = maps.b[1] = maps.out[0] = maps.out[1] = maps.a[0];  // what is not set below is not used
      if (dh && !few) {  // g (rows x vocab) times w (vocab x hidden, contiguous along hidden)
        Product& p = a.p[0];
        p.M = n;
        p.N = x.hidden;
        p.k_blocks = (int)((x.vocab + BK - 1) / BK);
        p.group = 8;
        if (int rc = map_16(&maps.b[0], x.w, x.hidden, x.vocab, x.ld_w, 64, FP16)) return rc;
        describe<FP16>(p, false, true);
        if (int rc = gradient_output<FP16>(maps, a, 0, dh_rows, b.partial_dh, nullptr, true, true, &join_dh)) return rc;
      }
      if (dw) {  // g^T (contiguous along vocab) times the hidden states (contiguous along hidden)
        Product& p = a.p[1];
        p.M = x.vocab;
        p.N = x.hidden;
        p.k_blocks = (int)((n + BK - 1) / BK);
        p.group = resident_group(2ll * TN * n);
        if (int rc = map_16(&maps.a[1], b.e, x.vocab, n, ld_e, 64, FP16)) return rc;
        if (int rc = map_16(&maps.b[1], b.h_copy, x.hidden, n, ld_copy, 64, FP16)) return rc;
        describe<FP16>(p, true, true);
        if (int rc = gradient_output<FP16>(maps, a, 1, dw, b.partial_dw, b.dw_sum, first, last, &join_dw)) return rc;
      }
      if (int rc = launch_product<kOut, FP16>(maps, a, x.stream)) return rc;
    }
    BiasSum bias = {};
    if (db) bias = BiasSum{b.bias_partial, db, b.scalars, x.vocab, row_blocks, !first, (int)((x.vocab + 31) / 32)};
    if (const int blocks = join_dh.blocks + join_dw.blocks + bias.blocks) {
      EVOX_CUDA(launch_overlapped(xent_join_kernel<FP16>, dim3((unsigned)blocks), 256, 0, 1, x.stream, join_dh, join_dw, bias));
    }
  }
  return EVOX_OK;
}

}  // namespace

int xent_finish(const float2* stats, long long ld_stats, const float* label_logit, const long long* labels, long long label_period,
                long long ignore_index, long long rows, long long vocab, float2* norm, float* loss, const int* status, cudaStream_t stream) {
  return finish(stats, ld_stats, label_logit, labels, label_period, ignore_index, rows, vocab, norm, loss, status, Weights{}, stream);
}

}  // namespace evox

using namespace evox;

extern "C" int32_t evox_linear_cross_entropy_copies(const void* h, int64_t ld_h, const void* w, int64_t ld_w) {
  return copies_of(h, ld_h, w, ld_w);
}

extern "C" size_t evox_linear_cross_entropy_workspace_bytes(int64_t rows, int64_t hidden, int64_t vocab, int32_t copies) {
  if (rows <= 0 || hidden <= 0 || vocab <= 0) return 0;
  Buffers b = {};
  return layout(b, nullptr, rows, hidden, vocab, copies, rows, false, false);
}

extern "C" int evox_linear_cross_entropy(const void* h, int64_t ld_h, const void* w, int64_t ld_w, int32_t dtype, const float* bias,
                                         const int64_t* labels, int64_t ignore_index, int64_t rows, int64_t hidden, int64_t vocab,
                                         int32_t reduction, float* loss, void* workspace, size_t workspace_bytes, int32_t* error_flag,
                                         void* stream) {
  if (int rc = check_operands("linear_cross_entropy", h, ld_h, w, ld_w, dtype, labels, rows, hidden, vocab, reduction, loss, workspace, error_flag))
    return rc;
  Buffers b = {};
  EVOX_REQUIRE(workspace_bytes >= layout(b, workspace, rows, hidden, vocab, copies_of(h, ld_h, w, ld_w), rows, false, false), EVOX_ERR_WORKSPACE,
               "linear_cross_entropy: workspace too small");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  Head x = {h, ld_h, w, ld_w, bias, (const long long*)labels, ignore_index, rows, hidden, vocab, error_flag, s};
  if (int rc = align_operands(x, b)) return rc;
  const bool per_row = reduction == EVOX_REDUCE_NONE, fp16 = dtype == EVOX_DTYPE_FP16;
  const Weights weights = {x.labels, rows, reduction, nullptr, 1.0f, per_row ? nullptr : b.scalars};
  float* row_loss = per_row ? loss : b.loss;
  if (b.few_logits) {
    if (int rc = fp16 ? few_loss_pass<true>(x, b, row_loss, weights) : few_loss_pass<false>(x, b, row_loss, weights)) return rc;
  } else {
    if (int rc = fp16 ? logits_pass<kLoss, true>(x, b, 0, rows, rows) : logits_pass<kLoss, false>(x, b, 0, rows, rows)) return rc;
    if (int rc = finish(b.stats, rows, b.label_logit, x.labels, rows, ignore_index, rows, vocab, nullptr, row_loss, x.error_flag, weights, s)) return rc;
  }
  if (!per_row) {
    EVOX_CUDA(launch_overlapped(xent_loss_sum_kernel, dim3(1), 256, 0, 1, s, b.loss, rows, b.scalars, loss));
  }
  return EVOX_OK;
}

extern "C" int64_t evox_linear_cross_entropy_chunk_rows(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0) return 0;
  // 2 GiB of exponentials at most (about 1 % of the memory), in whole tiles of rows
  const int64_t fit = (2ll << 30) / (up(vocab, 64) * 2) / TM * TM;
  const int64_t chunk = fit < TM ? TM : fit;
  return chunk < rows ? chunk : rows;
}

extern "C" size_t evox_linear_cross_entropy_grad_workspace_bytes(int64_t rows, int64_t hidden, int64_t vocab, int64_t chunk_rows,
                                                                 int32_t with_bias, int32_t copies) {
  if (rows <= 0 || hidden <= 0 || vocab <= 0 || chunk_rows <= 0) return 0;
  Buffers b = {};
  return layout(b, nullptr, rows, hidden, vocab, copies, chunk_rows < rows ? chunk_rows : rows, true, with_bias != 0);
}

extern "C" int evox_linear_cross_entropy_grad(const void* h, int64_t ld_h, const void* w, int64_t ld_w, int32_t dtype, const float* bias,
                                              const int64_t* labels, int64_t ignore_index, int64_t rows, int64_t hidden, int64_t vocab,
                                              int32_t reduction, const float* grad_loss, int64_t chunk_rows, float* loss, void* dh, void* dw,
                                              float* dbias, void* workspace, size_t workspace_bytes, int32_t* error_flag, void* stream) {
  if (int rc = check_operands("linear_cross_entropy_grad", h, ld_h, w, ld_w, dtype, labels, rows, hidden, vocab, reduction, loss, workspace, error_flag))
    return rc;
  EVOX_REQUIRE(chunk_rows > 0, EVOX_ERR_INVALID, "linear_cross_entropy_grad: chunk_rows must be positive");
  // the rescaling pass has a grid row per kRescaleColumns columns and two more; a grid has 65,535
  EVOX_REQUIRE(vocab <= 65533ll * kRescaleColumns, EVOX_ERR_INVALID, "linear_cross_entropy_grad: vocab must be at most %lld, got %lld",
               65533ll * kRescaleColumns, (long long)vocab);
  const long long chunk = chunk_rows < rows ? chunk_rows : rows;
  Buffers b = {};
  EVOX_REQUIRE(workspace_bytes >= layout(b, workspace, rows, hidden, vocab, copies_of(h, ld_h, w, ld_w), chunk, true, dbias != nullptr), EVOX_ERR_WORKSPACE,
               "linear_cross_entropy_grad: workspace too small");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  Head x = {h, ld_h, w, ld_w, bias, (const long long*)labels, ignore_index, rows, hidden, vocab, error_flag, s};
  if (int rc = align_operands(x, b)) return rc;
  return dtype == EVOX_DTYPE_FP16 ? gradient_pass<true>(x, b, chunk, reduction, grad_loss, loss, dh, dw, dbias)
                                  : gradient_pass<false>(x, b, chunk, reduction, grad_loss, loss, dh, dw, dbias);
}
