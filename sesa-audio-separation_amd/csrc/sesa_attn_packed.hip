// sesa_attention_packed: softmax attention within each sequence of a packed run, grouped heads, optional head gate.
//
// One pass over the keys with a running maximum and sum (fp32).  S^T = K Q^T on v_mfma_*_32x32x16: a lane then holds
// one query's scores, so the row statistics need a single exchange (the two lane halves), and the same registers,
// rounded to the type, are the second operand of O^T += V^T P^T; V^T comes from LDS by transposing 16-bit reads.
// Four waves of 32 queries share 64-key blocks of K and V in two LDS stages; blocks that every query of the tile sees run
// without masks, the diagonal and the last one apart.  Two (head 128) to four (head 64) workgroups a CU, out of step with
// each other, put one's softmax beside another's products: eight waves on one tile are slower (head 64 344 us where
// four take 311, head 128 412 and 381), two waves read K and V from LDS for half the queries (501 at head 128).
// Bound by the VALU about as much as by the matrix pipe: a 32 x 64 block is 32 exponentials and ~120 other operations
// a lane (~1000 cycles) against 512 (head 64) or 1024 (head 128) cycles of products.  Measured: 12289 causal tokens,
// 32 / 8 heads x 128, bf16 366-421 us by the sequences' lengths (0.92-1.05 PFLOP/s of its pairs; MFMA 53 % and VALU 52 %
// busy); 2 x 801 tokens x 62 lanes, 8 heads x 64, fp16 267-271 us (0.61 PFLOP/s: 13 blocks a tile, one of them masked, 89 %
// of the query rows used; MFMA 40 %, VALU 74 %).
// Probabilities are rounded to the 16-bit type for the product with v, which the matrix instructions take no wider: with the
// result's own rounding 2.9e-4 of it in fp16 and 2.0e-3 in bf16 against 64 bits (2.1e-4 and 1.6e-3 without).
#include "sesa_tokens.hpp"

namespace sesa {
namespace {

constexpr int kKeys = 64;   // keys per block

template <class T>
__device__ __forceinline__ f32x16 mfma16(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (std::is_same<T, f16>::value)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}

// Region i of the run: i = 0 the tokens before the first sequence, 1 .. n_seq the sequences, n_seq + 1 the rest.
__device__ __forceinline__ int64_t bound(const sesa_attn_args& a, int i) {
  if (i == 0) return 0;
  if (i == a.n_seq + 2) return a.tokens;
  if (!a.cu_seqlens) return (int64_t)(i - 1) * (a.tokens / a.n_seq);
  const int64_t c = a.cu_seqlens[i - 1];
  return c < 0 ? 0 : (c > a.tokens ? a.tokens : c);
}

// Query tiles: region i owns the slots bound(i) / BQ + i .. bound(i + 1) / BQ + i -- at least as many as its tiles of BQ
// tokens -- so a workgroup finds its tile from the boundaries alone (64 of them compared at a time), and the grid needs
// no count from the device.  The slots left over (less than one a region) end at once.
template <int BQ>
__device__ __forceinline__ bool find_tile(const sesa_attn_args& a, int slot, int* region, int* q0, int* start, int* end) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = a.n_seq + 2;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, i = lo + lane * step;
    const bool at = i < hi && bound(a, i) / BQ + i <= slot;
    const int c = max(1, (int)__popcll(__ballot(at)));
    lo += (c - 1) * step;
    hi = min(hi, lo + step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  const int64_t b = bound(a, lo), e = bound(a, lo + 1), q = b + (slot - (b / BQ + lo)) * (int64_t)BQ;
  *region = lo;
  *start = (int)b;
  *end = (int)e;
  *q0 = (int)q;
  return q >= b && q < e;
}

// kDma: rows of exactly D elements at 16-byte addresses, K and V go to LDS by global_load_lds_dwordx4 (no registers, no
// LDS stores; keys behind the sequence repeat its last one).  kDmaPart: the same for fewer elements, those behind head_dim
// zeroed once and their lanes kept out of the loads.  kRegisters: zeros behind the sequence and behind head_dim.
enum { kRegisters, kDma, kDmaPart };
template <class T, int D, int NW, int LOADS>
__global__ void __launch_bounds__(NW * 64, D == 64 ? (LOADS != kRegisters ? 4 : 3) : 2) attn_packed_kernel(sesa_attn_args a, int n_slots, int n_blocks_all) {
  constexpr bool DMA = LOADS != kRegisters, PART = LOADS == kDmaPart;
  constexpr int BQ = NW * 32, NTH = NW * 64, ROW = D * 2, IMG = kKeys * ROW, CH = D / 8, IT = kKeys * CH / NTH;
  constexpr float kLog2e = 1.4426950408889634f;
  __shared__ __attribute__((aligned(16))) char smem[4 * IMG];   // [stage][K, V], rows of D elements
  __shared__ int again;                                         // a row of the tile has to be done over
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hl = lane >> 5;
  const int group = a.heads / a.kv_heads;
  // a die's workgroups: consecutive query heads and tiles of one (lane, key head), so its L2 holds that head's K and V
  if (long_block() >= n_blocks_all) return;
  int t = die_tile((int)long_block(), n_blocks_all);
  const int gi = t % group;
  t /= group;
  const int slot = n_slots - 1 - t % n_slots;   // causal: the longest tiles first
  t /= n_slots;
  const int kh = t % a.kv_heads, ln = t / a.kv_heads;
  const int head = kh * group + gi;
  int region, q0, start, end;
  if (!find_tile<BQ>(a, slot, &region, &q0, &start, &end)) return;
  const int64_t q_pos = (int64_t)q0 + wave * 32 + l32;
  const bool q_ok = q_pos < end;
  T* out = reinterpret_cast<T*>(a.out) + q_pos * a.o_t + ln * a.o_l + head * a.o_h;
  if (region == 0 || region == a.n_seq + 1) {
    if (a.zero_rest && q_ok)
      for (int d = 8 * hl; d < a.head_dim; d += 16) store16(out + d, u32x4{0u, 0u, 0u, 0u});
    return;
  }
  if (tid == 0) again = 0;   // (set behind the barriers of the pass)
  const int hd = a.head_dim;
  const T* kp = reinterpret_cast<const T*>(a.k) + ln * a.k_l + kh * a.k_h;
  const T* vp = reinterpret_cast<const T*>(a.v) + ln * a.v_l + kh * a.v_h;

  u32x4 qf[D / 16];
  {
    const T* qp = reinterpret_cast<const T*>(a.q) + q_pos * a.q_t + ln * a.q_l + head * a.q_h;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int d = 16 * ks + 8 * hl;
      qf[ks] = q_ok && d < hd ? load16(qp + d) : u32x4{0u, 0u, 0u, 0u};
    }
  }
  f32x16 o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
  // Running reference r_run = a largest score so far times c (less kLift), rounded to fp32, and the running sum.  Every
  // probability is exp2(s c - r_run) with the product unrounded: the reference's own rounding is in all of them alike and cancels (a
  // product rounded anew for each use would not: 6e-2 of a block's weight at scores of 1e6).  From kFar on that rounding
  // may reach a factor of 2^0.5 and, further out, the range of P, so such rows are done over, where `sub` takes the maximum
  // off before the scaling: exactly 0 at the largest score, whatever its size.
  // kLift: fp16 takes P 2^7 higher, so that it is normal down to 2^-21 of the largest where plain P ends at 2^-14 (below,
  // a step is 2^-24: 100000 keys at 1.5 steps each lost a third of their weight).
  constexpr float kLift = std::is_same<T, f16>::value ? 7.f : 0.f;
  float r_run = -INFINITY, l_run = 0.f;
  const float c = a.scale * kLog2e;
  constexpr float kFar = 4194304.f;   // 2^22: fp32 steps of 2^-1
  bool far = false;

  // 16-byte chunk c of row r lies at c ^ key(r).  A K fragment read takes one chunk of 8 rows at a time, a transposing V
  // read four chunks of 4 rows: both sets fall into different banks (256 B of them: two rows of 64 elements, one of 128).
  auto key_of = [](int row) {
    return D == 64 ? ((row << 1) & 4) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3);
  };
  auto swz = [&](int row, int chunk) { return row * ROW + ((chunk ^ key_of(row)) << 4); };
  // DMA piece i of this wave: LDS bytes 1024 (wave + NW i) .. of an image, lane * 16 into it; the swizzle goes on the
  // source.  Offsets count from the block's first key.
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
  constexpr int PCS = IMG / 1024 / NW, RPP = 1024 / ROW;   // pieces per wave and image, rows per piece
  uint32_t koff[DMA ? PCS : 1], voff[DMA ? PCS : 1];
  uint32_t inside = 0;   // bit i: this lane's chunk of piece i lies inside head_dim (kDmaPart)
  auto lds_base = [](uint32_t v) { return PART ? (uint32_t)__builtin_amdgcn_readfirstlane(v) : v; };   // m0 inside a branch
  auto offsets = [&](int n) {   // n: keys of the block that exist
#pragma unroll
    for (int i = 0; i < PCS; ++i) {
      const int row = (wave + NW * i) * RPP + lane / CH, ch = (lane % CH) ^ key_of(row), r = min(row, n - 1);
      if constexpr (PART) inside |= (uint32_t)(ch * 8 < hd) << i;
      koff[i] = (uint32_t)(r * (int)a.k_t + ch * 8) * 2u;
      voff[i] = (uint32_t)(r * (int)a.v_t + ch * 8) * 2u;
    }
  };
  u32x4 kreg[DMA ? 1 : IT], vreg[DMA ? 1 : IT];
  auto load_block = [&](int kb, int stage) {
    const int64_t p0 = (int64_t)start + kb * kKeys;
    if constexpr (DMA) {
      if (p0 + kKeys > end) offsets((int)(end - p0));
      const char* kb0 = reinterpret_cast<const char*>(kp + p0 * a.k_t);
      const char* vb0 = reinterpret_cast<const char*>(vp + p0 * a.v_t);
#pragma unroll
      for (int i = 0; i < PCS; ++i)
        if (!PART || (inside >> i & 1)) dma16_asm(kb0, koff[i], lds_base(lds0 + stage + (wave + NW * i) * 1024));
#pragma unroll
      for (int i = 0; i < PCS; ++i)
        if (!PART || (inside >> i & 1)) dma16_asm(vb0, voff[i], lds_base(lds0 + stage + IMG + (wave + NW * i) * 1024));
    } else {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int e = tid + i * NTH, d = e % CH * 8;
        const int64_t p = p0 + e / CH;
        const bool ok = p < end && d < hd;
        kreg[i] = ok ? load16(kp + p * a.k_t + d) : u32x4{0u, 0u, 0u, 0u};
        vreg[i] = ok ? load16(vp + p * a.v_t + d) : u32x4{0u, 0u, 0u, 0u};
      }
    }
  };
  auto store_block = [&](int stage) {
    if constexpr (!DMA) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int e = tid + i * NTH, off = swz(e / CH, e % CH);
        *reinterpret_cast<u32x4*>(smem + stage + off) = kreg[i];
        *reinterpret_cast<u32x4*>(smem + stage + IMG + off) = vreg[i];
      }
    }
  };
  // Fragment addresses: a key block's K row 32 rb + l32 and V rows 16 ks + .. differ from the first ones' by whole
  // multiples of 16 rows, which leave key_of alone, so one offset per chunk serves all of them.
  // V^T (d-block db, keys 16 ks ..): lane half hl gets the keys 4 hl .. + 3 and 8 + 4 hl .. + 3 of its step, the order in
  // which the score registers hold them.
  typedef __attribute__((address_space(3))) char lds_char;
  typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
  lds_char* const lds = (lds_char*)smem;
  int ko[D / 16], vo[2][D / 32];
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) ko[ks] = swz(l32, 2 * ks + hl);
  {
    const int tg = lane >> 4, ti = lane & 15, key = 4 * (tg >> 1) + (ti >> 2);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      const int d = db * 32 + 16 * (tg & 1) + 4 * (ti & 3);
      vo[0][db] = IMG + swz(key, d >> 3) + ((d & 7) << 1);
      vo[1][db] = IMG + swz(key + 8, d >> 3) + ((d & 7) << 1);
    }
  }
  auto vt = [&](int stage, int ks, int db) -> u32x4 {   // (16-bit elements move through the read unchanged)
    const bf16x4 t0 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (__attribute__((address_space(3))) bf16x4*)(lds + stage + vo[0][db] + 16 * ROW * ks));
    const bf16x4 t1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
        (__attribute__((address_space(3))) bf16x4*)(lds + stage + vo[1][db] + 16 * ROW * ks));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(t0, t1, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  const int last = a.causal ? min(end, q0 + BQ) : end;   // keys from here on reach no query of the tile
  const int n_blocks = (last - start + kKeys - 1) / kKeys;
  // blocks all of whose keys every query of the tile sees
  const int n_whole = (min(end, a.causal ? q0 + 1 : end) - start) / kKeys;

  // Second pass (REDO): infinite and NaN elements of v are taken out, so that a probability of 0 -- a key that the row does
  // not see, or one too small for the type -- times one of them is no NaN, and come back as what the keys that the row does
  // see make of them.  code: 1 for +inf, 128 for -inf, 16384 for NaN; 16 keys' codes add up without a carry.
  auto take_out = [](u32x4& v, u32x4& code) {
    constexpr bool F16 = std::is_same<T, f16>::value;
    constexpr uint32_t kExp = F16 ? 0x7c00 : 0x7f80, kFrac = F16 ? 0x03ff : 0x007f;
    constexpr uint32_t kPos = F16 ? 0x3c00 : 0x3f80, kNeg = F16 ? 0x5800 : 0x4300, kNan = F16 ? 0x7400 : 0x4680;
    bool any = false;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t keep = 0, out = 0;
#pragma unroll
      for (int h = 0; h < 32; h += 16) {
        const uint32_t e = v[q] >> h & 0xffffu;
        const bool bad = (e & kExp) == kExp;
        any = any || bad;
        keep |= (bad ? 0u : e) << h;
        out |= (!bad ? 0u : e & kFrac ? kNan : e >> 15 ? kNeg : kPos) << h;
      }
      v[q] = keep;
      code[q] = out;
    }
    return any;
  };
  // A finite score never weighs less than this in the second pass, nor does a rescaling: too little to move a finite sum; an
  // infinite one stays what it is, and p > 0 says which keys the row sees.
  constexpr float kLeast = 1.17549435e-38f;   // 2^-126

  auto step = [&](int kb, auto masked, auto second) {
    constexpr bool MASKED = decltype(masked)::value, REDO = decltype(second)::value;
    const int cur = (kb & 1) * 2 * IMG, next = ((kb + 1) & 1) * 2 * IMG;
    // this wave's part of block kb has landed; behind the barrier everyone's has, and everyone is done with block
    // kb - 1, whose place block kb + 1 takes
    if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    sesa_sync();
    if (kb + 1 < n_blocks) load_block(kb + 1, next);
    f32x16 s[2];
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      u32x4 kf[D / 16];
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) kf[ks] = *(__attribute__((address_space(3))) const u32x4*)(lds + cur + ko[ks] + rb * 32 * ROW);
      __builtin_amdgcn_sched_barrier(0);   // all reads before the first product: one LDS round trip, not one a product
#pragma unroll
      for (int r = 0; r < 16; ++r) s[rb][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) s[rb] = mfma16<T>(kf[ks], qf[ks], s[rb]);
    }
    // last key of the block that this query sees, counted like the registers' keys (4 hl taken off)
    const int lim = (int)min((int64_t)(end - 1), a.causal ? q_pos : (int64_t)(end - 1)) - (start + kb * kKeys) - 4 * hl;
    if constexpr (MASKED) {
#pragma unroll
      for (int rb = 0; rb < 2; ++rb)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (rb * 32 + (r & 3) + 8 * (r >> 2) > lim) s[rb][r] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[rb][r]);
    top = max_halves(top);
    // The reference moves only when a block exceeds it by more than 2^8 in the exponential (P stays below 2^(8.5 + kLift), in
    // range for fp16), so most blocks leave O alone.  Both halves of a query hold the same values, so they agree.
    const bool raw = REDO && far;   // r_run holds the score itself
    if ((raw ? (top - r_run) * c + kLift : fmaf(top, c, -r_run)) > 8.f + kLift) {
      const float r = raw ? top : fmaf(top, c, -kLift);
      float alpha = __builtin_amdgcn_exp2f(raw ? (r_run - r) * c : r_run - r);   // (the first time: 0)
      if constexpr (REDO) alpha = fmaxf(alpha, kLeast);
      else far = far || (fabsf(top) < INFINITY && !(fabsf(r) <= kFar));
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] *= alpha;
      r_run = r;
    }
    float rc = r_run == -INFINITY ? 0.f : r_run, sub = 0.f;   // (no finite score so far: every P is exp(-inf) = 0)
    if (raw) sub = rc, rc = -kLift;
    float sum[2] = {0.f, 0.f};   // a block's own first: small ones would be lost one by one against a large l_run
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float p = __builtin_amdgcn_exp2f(fmaf(REDO ? s[rb][r] - sub : s[rb][r], c, -rc));
        if (REDO && p < kLeast && s[rb][r] > -INFINITY) p = kLeast;
        s[rb][r] = p;
        sum[rb] += p;
      }
    l_run += sum[0] + sum[1];   // this half's keys; the halves join at the end
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      f32x16& sv = s[ks >> 1];
      const int r0 = 8 * (ks & 1);
      const u32x4 pf = {pack2t<T>(sv[r0], sv[r0 + 1]), pack2t<T>(sv[r0 + 2], sv[r0 + 3]), pack2t<T>(sv[r0 + 4], sv[r0 + 5]),
                        pack2t<T>(sv[r0 + 6], sv[r0 + 7])};
      u32x4 vf[D / 32];
#pragma unroll
      for (int db = 0; db < D / 32; ++db) vf[db] = vt(cur, ks, db);
      if constexpr (REDO) {
        u32x4 seen;
#pragma unroll
        for (int q = 0; q < 4; ++q) seen[q] = pack2t<T>(sv[r0 + 2 * q] > 0.f ? 1.f : 0.f, sv[r0 + 2 * q + 1] > 0.f ? 1.f : 0.f);
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
          u32x4 code;
          if (__ballot(take_out(vf[db], code))) {
            f32x16 n;
#pragma unroll
            for (int r = 0; r < 16; ++r) n[r] = 0.f;
            n = mfma16<T>(code, seen, n);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int k = (int)n[r];
              o[db][r] += (k >= 16384 ? __builtin_nanf("") : 0.f) + ((k & 16383) >= 128 ? -INFINITY : 0.f) + (k & 127 ? INFINITY : 0.f);
            }
          }
        }
      }
#pragma unroll
      for (int db = 0; db < D / 32; ++db) o[db] = mfma16<T>(vf[db], pf, o[db]);
    }
    if (kb + 1 < n_blocks) store_block(next);
  };

  if constexpr (DMA) {
    offsets(min(kKeys, end - start));
    if constexpr (PART) {
      for (int e = tid * 16; e < 4 * IMG; e += NTH * 16) *reinterpret_cast<u32x4*>(smem + e) = u32x4{0u, 0u, 0u, 0u};
      sesa_sync();
    }
  }
  load_block(0, 0);
  store_block(0);
  __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0), where the compiler sees it: no wait for Q inside the loop
  int kb = 0;
  for (; kb < n_whole; ++kb) step(kb, std::false_type{}, std::false_type{});
  for (; kb < n_blocks; ++kb) step(kb, std::true_type{}, std::false_type{});
  l_run += __shfl_xor(l_run, 32);

  // Rows to do over: `far`, and NaN in o under finite probabilities (0 times an infinite or NaN v, an infinity times a
  // rescaling by 0; NaN scores make the sum NaN as well: that row is NaN by the formula).  Nothing to look for inside the
  // loop.  The whole tile goes through its keys once more, with the elements taken out (2 x 801 tokens x 62 lanes, every tile:
  // 267 -> 734 us; 12289 causal tokens, scores of 1e9 in every row: 0.4 -> 1.3 ms; a serial pass over a row's keys instead
  // took 10 and 69 ms); rows that did not ask for it come out as they were.
  bool over = false;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) over = over || o[db][r] != o[db][r];
  over = q_ok && (far || (over && l_run == l_run));
  if (__ballot(over) && lane == 0) again = 1;
  sesa_sync();
  if (__builtin_amdgcn_readfirstlane(again)) {
    r_run = -INFINITY;
    l_run = 0.f;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
    if constexpr (DMA) offsets(min(kKeys, end - start));
    load_block(0, 0);
    store_block(0);
#pragma unroll 1
    for (kb = 0; kb < n_blocks; ++kb) step(kb, std::true_type{}, std::true_type{});
    l_run += __shfl_xor(l_run, 32);
  }

  if (!q_ok) return;
  float scale = 1.f / l_run;
  if (a.gate) scale *= sigmoid_f((float)reinterpret_cast<const T*>(a.gate)[q_pos * a.g_t + ln * a.g_l + head * a.g_h]);
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const int d = db * 32 + 8 * b + 4 * hl;
      if (d >= hd) continue;
      struct __attribute__((packed)) B8 { uint32_t a, b; };
      *reinterpret_cast<B8*>(out + d) = B8{pack2t<T>(o[db][4 * b] * scale, o[db][4 * b + 1] * scale),
                                           pack2t<T>(o[db][4 * b + 2] * scale, o[db][4 * b + 3] * scale)};
    }
}

template <class T>
int launch_attn(const sesa_attn_args& a, hipStream_t st) {
  constexpr int NW = 4;
  const int64_t n_slots = a.tokens / (NW * 32) + a.n_seq + 2;
  const int64_t blocks = n_slots * a.heads * a.lanes;
  SESA_REQUIRE(blocks < (1ll << 31), SESA_ERR_INVALID, "attention_packed: too many tokens x heads x lanes");
  // 16-byte rows, and a block's byte offsets in 32 bits (12289 causal tokens, 32 / 8 heads, bf16, aligned | through registers:
  // 64 181 | 224 us, 96 286 | 361, 128 298 | 400).  Rows of the whole tile width have a kernel of their own: the part rows'
  // masks take 4 % there.
  const int64_t strides = a.k_t | a.k_l | a.k_h | a.v_t | a.v_l | a.v_h;
  const bool dma = strides % 8 == 0 && ((uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0 && a.k_t >= 0 && a.v_t >= 0 &&
                   a.k_t < (1 << 23) && a.v_t < (1 << 23);
  const dim3 grid = long_grid(blocks), block(NW * 64);
  const int nb = (int)blocks;
  if (a.head_dim <= 64) {
    if (!dma) hipLaunchKernelGGL((attn_packed_kernel<T, 64, NW, kRegisters>), grid, block, 0, st, a, (int)n_slots, nb);
    else if (a.head_dim == 64) hipLaunchKernelGGL((attn_packed_kernel<T, 64, NW, kDma>), grid, block, 0, st, a, (int)n_slots, nb);
    else hipLaunchKernelGGL((attn_packed_kernel<T, 64, NW, kDmaPart>), grid, block, 0, st, a, (int)n_slots, nb);
  } else {
    if (!dma) hipLaunchKernelGGL((attn_packed_kernel<T, 128, NW, kRegisters>), grid, block, 0, st, a, (int)n_slots, nb);
    else if (a.head_dim == 128) hipLaunchKernelGGL((attn_packed_kernel<T, 128, NW, kDma>), grid, block, 0, st, a, (int)n_slots, nb);
    else hipLaunchKernelGGL((attn_packed_kernel<T, 128, NW, kDmaPart>), grid, block, 0, st, a, (int)n_slots, nb);
  }
  SESA_CHECK_LAUNCH();
  return SESA_OK;
}

}  // namespace
}  // namespace sesa

using namespace sesa;

extern "C" int sesa_attention_packed(const sesa_attn_args* args, void* stream) {
  clear_error();
  SESA_REQUIRE(args, SESA_ERR_INVALID, "attention_packed: null arguments");
  const sesa_attn_args& a = *args;
  SESA_REQUIRE(a.tokens >= 0 && a.tokens < (1ll << 31) - 1024, SESA_ERR_INVALID, "attention_packed: tokens %lld",
               (long long)a.tokens);
  SESA_REQUIRE(a.lanes >= 1 && a.heads >= 1 && a.kv_heads >= 1 && a.heads % a.kv_heads == 0, SESA_ERR_INVALID,
               "attention_packed: lanes %d, heads %d, kv_heads %d", a.lanes, a.heads, a.kv_heads);
  SESA_REQUIRE(a.head_dim >= 8 && a.head_dim <= 128 && a.head_dim % 8 == 0, SESA_ERR_INVALID,
               "attention_packed: head_dim %d (a multiple of 8, 8..128)", a.head_dim);
  SESA_REQUIRE(a.dtype == SESA_DTYPE_F16 || a.dtype == SESA_DTYPE_BF16, SESA_ERR_INVALID, "attention_packed: dtype %d",
               a.dtype);
  SESA_REQUIRE(a.n_seq >= 1 && a.n_seq < (1 << 30), SESA_ERR_INVALID, "attention_packed: n_seq %d", a.n_seq);
  SESA_REQUIRE(a.cu_seqlens || a.tokens % a.n_seq == 0, SESA_ERR_INVALID,
               "attention_packed: %lld tokens are not %d sequences of one length", (long long)a.tokens, a.n_seq);
  SESA_REQUIRE(a.scale > 0.f && a.scale < INFINITY, SESA_ERR_INVALID, "attention_packed: scale %g", (double)a.scale);
  if (a.tokens == 0) return SESA_OK;
  SESA_REQUIRE(a.q && a.k && a.v && a.out, SESA_ERR_INVALID, "attention_packed: null operand");
  hipStream_t st = as_stream(stream);
  return a.dtype == SESA_DTYPE_F16 ? launch_attn<f16>(a, st) : launch_attn<__bf16>(a, st);
}
