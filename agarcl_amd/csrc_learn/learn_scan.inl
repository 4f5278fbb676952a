// learn_scan.inl -- linear recurrences y[t] = a[t] y[t-1] + b[t] over the steps of a rollout, for many columns at once.
//
// A segment is 8 steps (AGARCL_MARK_STEPS).  One thread owns a segment of VEC neighbouring columns: it loads the segment into registers and works out, step by
// step, y[i] = P[i] y + B[i] over the y that enters -- before it knows that y.  A workgroup is CL column lanes x TL = 256 / CL time lanes and takes TL segments in
// a row at once: the segments' maps are joined over the time lanes of a wavefront by shuffles and over the wavefronts through LDS, with one barrier per TL
// segments, and then every step is one multiplication and addition away.  The next segment's loads are under way meanwhile.  Column lanes are the fast index
// of a wavefront, so its loads are runs of CL x VEC elements.  Where there are too few columns to fill the chip the steps are cut into chunks as well: a
// first launch leaves every chunk's map, the second starts each chunk from the maps in front of it.
//
// A map's P is 0 exactly where a step of it drops what came before (a reset, the end of an episode): joining looks at P and never multiplies what was
// dropped, so infinities and NaN do not pass.  A product of gates is kept from underflowing to 0 (times 1e-38 is nothing in 32 bits all the same).

// VEC neighbouring elements as they were loaded: 16-bit ones stay two to a register
template <class T, int VEC> struct Raw {
  uint32_t w[(VEC * sizeof(T) + 3) / 4];
  __device__ __forceinline__ float operator[](int j) const;
  __device__ __forceinline__ void all(T v) {
    uint32_t b;
    if constexpr (sizeof(T) == 4) b = __builtin_bit_cast(uint32_t, v);
    else b = __builtin_bit_cast(uint16_t, v) * 0x10001u;
#pragma unroll
    for (auto &r : w) r = b;
  }
  // a later use takes the registers from here on: keeps the compiler from holding what it derived from them in twice as many
  __device__ __forceinline__ void anew() {
#pragma unroll
    for (auto &r : w) asm volatile("" : "+v"(r));
  }
};
template <class T, int VEC> __device__ __forceinline__ float Raw<T, VEC>::operator[](int j) const {
  if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
  else if constexpr (std::is_same<T, bf16_t>::value) return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
  else return (float)__builtin_bit_cast(f16_t, (uint16_t)(w[j / 2] >> (16 * (j & 1))));
}
// (aligned as an element is, no more: the hardware takes wide loads at any address)
template <class T, int VEC> struct __attribute__((packed, aligned(alignof(T)))) Pack { T v[VEC]; };

template <class T, int VEC> __device__ __forceinline__ void load_raw(Raw<T, VEC> &out, const T *p) {
  out.w[(VEC * sizeof(T) - 1) / 4] = 0;
  __builtin_memcpy(out.w, (const Pack<T, VEC> *)p, VEC * sizeof(T));
}
template <int VEC> __device__ __forceinline__ void load_floats(float (&out)[VEC], const float *p) {
  Raw<float, VEC> r; load_raw<float, VEC>(r, p);
#pragma unroll
  for (int j = 0; j < VEC; ++j) out[j] = r[j];
}
template <class T, int VEC> __device__ __forceinline__ void store_pack(T *p, const float (&in)[VEC]) {
  Pack<T, VEC> k;
#pragma unroll
  for (int j = 0; j < VEC; ++j) k.v[j] = from_f<T>(in[j]);
  *(Pack<T, VEC> *)p = k;
}
template <int VEC> struct Map { float P[VEC], B[VEC]; };
__device__ __forceinline__ float map_at(float P, float B, float y) { return P == 0.f ? B : fmaf(P, y, B); }
__device__ __forceinline__ float map_p(float a, float b) { return a == 0.f || b == 0.f ? 0.f : fmaxf(a * b, 1.17549435e-38f); }
template <int VEC> __device__ __forceinline__ void map_clear(Map<VEC> &m) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) { m.P[j] = 1.f; m.B[j] = 0.f; }
}
// first e, then m
template <int VEC> __device__ __forceinline__ void map_behind(Map<VEC> &m, const Map<VEC> &e) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) { m.B[j] = map_at(m.P[j], m.B[j], e.B[j]); m.P[j] = map_p(m.P[j], e.P[j]); }
}

static const int SEG = AGARCL_MARK_STEPS;

// the shape of a launch: chosen on the host (scan_shape)
struct ScanShape { int cl_log, chunks; int64_t steps, segments, chunk_segments, columns, groups, slots; };      // slots: groups, up to a multiple of 8

template <int VEC> struct ScanLds { Map<VEC> total[2][256]; };   // [parity][wavefront (or pair, or all four) x column lane]

// this thread's place
struct ScanLane { int cl, col, tl, tls, in_wave, units, unit; };
__device__ __forceinline__ ScanLane scan_lane(int cl_log) {
  ScanLane s; s.cl = 1 << cl_log; s.col = threadIdx.x & (s.cl - 1); s.tl = threadIdx.x >> cl_log; s.tls = 256 >> cl_log;
  const int unit_log = cl_log > 6 ? cl_log : 6;
  s.in_wave = 64 >> cl_log; s.unit = threadIdx.x >> unit_log; s.units = 256 >> unit_log;
  return s;
}

// from this thread's map: what all time lanes before it make together (before), and all of them (all), for its columns
template <int VEC> __device__ __forceinline__ void scan_join(const ScanLane &s, Map<VEC> m, Map<VEC> &before, Map<VEC> &all, ScanLds<VEC> &lds, int parity) {
  const int lane = threadIdx.x & 63;
  for (int d = s.cl; d < 64; d <<= 1) {
    Map<VEC> e;
#pragma unroll
    for (int j = 0; j < VEC; ++j) { e.P[j] = __shfl_up(m.P[j], d); e.B[j] = __shfl_up(m.B[j], d); }
    if (lane >= d) map_behind(m, e);
  }
  map_clear(before);
  if (s.in_wave > 1) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float P = __shfl_up(m.P[j], s.cl), B = __shfl_up(m.B[j], s.cl);
      if (lane >= s.cl) { before.P[j] = P; before.B[j] = B; }
    }
  }
  if (s.in_wave <= 1 || lane >= 64 - s.cl) lds.total[parity][s.unit * s.cl + s.col] = m;
  __syncthreads();
  Map<VEC> front; map_clear(front); map_clear(all);
  for (int u = 0; u < s.units; ++u) {
    if (u == s.unit) front = all;
    Map<VEC> t = lds.total[parity][u * s.cl + s.col];
    map_behind(t, all); all = t;
  }
  map_behind(before, front);
}

// Where a thread's segment lies: step t0 of the rollout, `t` steps behind step `base`, which is the same for the workgroup; its columns are `c` behind column
// `cbase`.  n: how many of its 8 steps there are (0: the thread has no segment in this turn).
struct Place { int64_t base, cbase; uint32_t t, c; int n; };
// An array of steps x columns is read and written through a buffer descriptor per step: the base is the step's (scalar), the offset is the thread's, 32 bits (they
// fit: see scan_shape).  A step that is not there has an offset behind the descriptor's 2^31 bytes, and an array that is not there has a descriptor of none: such a
// load gives 0 and such a store is dropped.  So a turn has no branch around its loads and stores, and the compiler can count how many are under way -- with
// branches it waited for all of them, the stores of the turn before too (256 x 4096 x 64 bf16, 2^8 lanes: forward 94 us with branches, 89 without, gradient 161 and 147;
// and a sixth fewer registers).
static const uint32_t kGone = 0x80000000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t span(uintptr_t at, bool some) { return __builtin_amdgcn_make_buffer_rsrc((void *)at, 0, some ? kGone : 0, 0x00020000); }
template <class T> struct Rows {
  uintptr_t p; int64_t stride;
  __device__ __forceinline__ uint32_t offset(const Place &w) const { return (w.t * (uint32_t)stride + w.c) * (uint32_t)sizeof(T); }
  __device__ __forceinline__ uintptr_t first(const Place &w) const { return p + (w.base * stride + w.cbase) * (int64_t)sizeof(T); }      // the same for the workgroup
  __device__ __forceinline__ int64_t step() const { return stride * (int64_t)sizeof(T); }
};
__device__ __forceinline__ uint32_t if_there(uint32_t off, bool there) { return there ? off : kGone; }
template <class T, int VEC> __device__ __forceinline__ void fetch(Raw<T, VEC> &out, __amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (VEC * sizeof(T) == 2) out.w[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
  else if constexpr (VEC * sizeof(T) == 4) out.w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
  else { const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0); out.w[0] = v[0]; out.w[1] = v[1]; }
}
template <class T, int VEC> __device__ __forceinline__ void put(__amdgpu_buffer_rsrc_t r, uint32_t off, const float (&in)[VEC]) {
  Pack<T, VEC> k;
#pragma unroll
  for (int j = 0; j < VEC; ++j) k.v[j] = from_f<T>(in[j]);
  if constexpr (VEC * sizeof(T) == 2) __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, k), r, off, 0, 0);
  else if constexpr (VEC * sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, k), r, off, 0, 0);
  else { typedef uint32_t u32x2 __attribute__((ext_vector_type(2))); __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, k), r, off, 0, 0); }
}

// Op: load(place) -> registers; prep(Map &): what can be known without the y that enters; write(place, y).  Op::reverse: the last segment is first.
// work: [2][chunks][columns] maps of the chunks.  MAPS leaves them, CHUNK begins where they lead, WHOLE is a launch without chunks: a kernel of its own, since the
// registers that the joining of the maps takes would cost it a wavefront per SIMD.
enum { WHOLE, MAPS, CHUNK };
template <class Op, int VEC, int MODE>
__device__ __forceinline__ void scan_columns(Op &op, const ScanShape &sh, const float *start, float *end, float *work, ScanLds<VEC> &lds) {
  const ScanLane s = scan_lane(sh.cl_log);
  int parity = 0;
  const int64_t q = blockIdx.y, first = q * sh.chunk_segments, stop = first + sh.chunk_segments < sh.segments ? first + sh.chunk_segments : sh.segments;
  for (int64_t b = blockIdx.x; b < sh.slots; b += gridDim.x) {
    // neighbouring column groups share 128-byte lines where they are narrow: keep them on one XCD, behind one L2 (workgroups go to the 8 XCDs in turn)
    const int64_t group = sh.slots >= 16 ? (b & 7) * (sh.slots >> 3) + (b >> 3) : b;
    if (group >= sh.groups) continue;
    int64_t cbase = (group << sh.cl_log) * VEC, c0 = cbase + s.col * VEC;
    const bool there = c0 < sh.columns;
    // (the last thread of a row of columns that VEC does not divide takes some of its neighbour's, too, and writes the same there; where it is its workgroup's
    // first, the workgroup begins there, or the offset from its beginning would be below 0)
    if (cbase + VEC > sh.columns) cbase = sh.columns - VEC;
    if (there && c0 + VEC > sh.columns) c0 = sh.columns - VEC;
    op.start(cbase, there ? c0 : cbase);
    // the turn that begins with segment k0 (counted in the scan's order)
    const auto place = [&](int64_t k0) __attribute__((always_inline)) {
      const int64_t low = sh.segments - s.tls - k0, base = Op::reverse ? (low > 0 ? low : 0) : k0, at = Op::reverse ? sh.segments - 1 - k0 - s.tl : k0 + s.tl;
      const bool on = k0 + s.tl < stop && there;
      const int64_t left = sh.steps - at * SEG;
      return Place{base * SEG, cbase, on ? (uint32_t)(at - base) * SEG : 0u, there ? (uint32_t)(c0 - cbase) : 0u, on ? (left < SEG ? (int)left : SEG) : 0};
    };
    float y[VEC];
    Map<VEC> run; map_clear(run);
    if (MODE != MAPS) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) y[j] = start && there ? start[c0 + j] : 0.f;
    }
    op.load(place(first));
    if (MODE == CHUNK && q) {      // the chunks in front: each time lane joins a part of their maps, then all of them
      const int64_t each = (q + s.tls - 1) / s.tls, lo = s.tl * each, hi = lo + each < q ? lo + each : q;
      Map<VEC> f, before, all; map_clear(f);
      for (int64_t c = lo; c < hi; c += 2) {
        Map<VEC> t[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          map_clear(t[i]);
          if (c + i < hi && there) {
            const float *p = work + (c + i) * sh.columns + c0;
            load_floats<VEC>(t[i].P, p); load_floats<VEC>(t[i].B, p + sh.chunks * sh.columns);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) { map_behind(t[i], f); f = t[i]; }
      }
      scan_join(s, f, before, all, lds, parity); parity ^= 1;
#pragma unroll
      for (int j = 0; j < VEC; ++j) y[j] = map_at(all.P[j], all.B[j], y[j]);
    }
    if (MODE != MAPS) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) asm volatile("" : "+v"(y[j]));      // (waited for here, or every turn would wait for all the loads that are under way)
    }
    for (int64_t k0 = first; k0 < stop; k0 += s.tls) {
      Map<VEC> m;
      map_clear(m);
      if (k0 + s.tl < stop && there) op.prep(m);
      if (k0 + s.tls < stop) op.load(place(k0 + s.tls));      // (under way while the maps are joined and the steps written)
      float e[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) e[j] = MODE == MAPS ? 0.f : y[j];
      if (MODE == MAPS || s.tls > 1) {
        Map<VEC> before, all;
        scan_join(s, m, before, all, lds, parity); parity ^= 1;
        if (MODE == MAPS) { map_behind(all, run); run = all; }
        else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) { e[j] = map_at(before.P[j], before.B[j], y[j]); y[j] = map_at(all.P[j], all.B[j], y[j]); }
        }
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = map_at(m.P[j], m.B[j], y[j]);
      }
      if (MODE != MAPS) op.write(place(k0), e);
    }
    if (s.tl == 0 && there) {
      if (MODE == MAPS) { store_pack<float, VEC>(work + q * sh.columns + c0, run.P); store_pack<float, VEC>(work + (sh.chunks + q) * sh.columns + c0, run.B); }
      else if (end && stop == sh.segments) store_pack<float, VEC>(end + c0, y);
    }
  }
}
