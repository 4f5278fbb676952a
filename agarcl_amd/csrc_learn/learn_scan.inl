// learn_scan.inl -- linear recurrences y[t] = a[t] y[t-1] + b[t] over the steps of a rollout, for many columns at once.
//
// A segment is 8 steps (AGARCL_MARK_STEPS).  One thread owns a segment of VEC neighbouring columns: it loads the segment once into registers, works out the
// segment's own map y -> P y + B, and -- when it knows the y that enters -- goes through the steps again from registers and writes.  A workgroup is CL column
// lanes x TL = 256 / CL time lanes and takes TL segments in a row at once: the maps are joined over the time lanes of a wavefront by shuffles and over the
// wavefronts through LDS, with one barrier per TL segments.  Column lanes are the fast index of a wavefront, so its loads are runs of CL x VEC elements.
// Where there are too few columns to fill the chip the steps are cut into chunks as well: a first launch leaves every chunk's map, the second starts each chunk
// from the maps in front of it.
//
// A map's P is 0 exactly where a step of it drops what came before (a reset, the end of an episode): joining looks at P and never multiplies what was
// dropped, so infinities and NaN do not pass.  A product of gates is kept from underflowing to 0 (times 1e-38 is nothing in 32 bits all the same).
// VEC neighbouring elements as they were loaded: 16-bit ones stay two to a register
template <class T, int VEC> struct Raw {
  uint32_t w[(VEC * sizeof(T) + 3) / 4];
  __device__ __forceinline__ float operator[](int j) const;
  // a later use takes the registers from here on: keeps the compiler from holding what it derived from them (a gate's sigmoids) in twice as many
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

template <class T, int VEC> __device__ __forceinline__ void load_raw(Raw<T, VEC> &out, const T *p, int nv) {
  if constexpr (VEC * sizeof(T) < 4) { out.w[0] = nv ? (uint32_t)*(const uint16_t *)p : 0u; }
  else {
    if (nv == VEC) __builtin_memcpy(out.w, (const Pack<T, VEC> *)p, VEC * sizeof(T));
    else {
#pragma unroll
      for (int k = 0; k < (int)(VEC * sizeof(T) / 4); ++k) {
        if constexpr (sizeof(T) == 4) out.w[k] = k < nv ? ((const uint32_t *)p)[k] : 0u;
        else out.w[k] = (2 * k < nv ? (uint32_t)((const uint16_t *)p)[2 * k] : 0u) | (2 * k + 1 < nv ? (uint32_t)((const uint16_t *)p)[2 * k + 1] << 16 : 0u);
      }
    }
  }
}
template <int VEC> __device__ __forceinline__ void load_floats(float (&out)[VEC], const float *p, int nv) {
  Raw<float, VEC> r; load_raw<float, VEC>(r, p, nv);
#pragma unroll
  for (int j = 0; j < VEC; ++j) out[j] = r[j];
}
template <class T, int VEC> __device__ __forceinline__ void store_pack(T *p, const float (&in)[VEC], int nv) {
  Pack<T, VEC> k;
#pragma unroll
  for (int j = 0; j < VEC; ++j) k.v[j] = from_f<T>(in[j]);
  if (nv == VEC) *(Pack<T, VEC> *)p = k;
  else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) if (j < nv) p[j] = k.v[j];
  }
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

// the shape of a launch: chosen on the host (scan_plan)
struct ScanShape { int cl_log, chunks; int64_t segments, chunk_segments, columns, groups; };

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

// Op: load(segment) -> registers, map(Map &), run(segment, float (&y)[VEC]) goes through the steps from y and writes.  Op::reverse: the last segment is first.
// work: [2][chunks][columns] maps of the chunks
template <class Op, int VEC, bool MAPS>
__device__ __forceinline__ void scan_columns(Op &op, const ScanShape &sh, const float *start, float *end, float *work, ScanLds<VEC> &lds) {
  const ScanLane s = scan_lane(sh.cl_log);
  int parity = 0;
  const int64_t q = blockIdx.y, first = q * sh.chunk_segments, stop = first + sh.chunk_segments < sh.segments ? first + sh.chunk_segments : sh.segments;
  for (int64_t group = blockIdx.x; group < sh.groups; group += gridDim.x) {
    const int64_t c0 = ((group << sh.cl_log) + s.col) * VEC;
    const int nv = c0 >= sh.columns ? 0 : sh.columns - c0 < VEC ? (int)(sh.columns - c0) : VEC;
    op.place(c0, nv);
    float y[VEC];
    Map<VEC> run; map_clear(run);
    if (!MAPS) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) y[j] = start && j < nv ? start[c0 + j] : 0.f;
      if (q) {      // the chunks in front: each time lane joins a part of their maps, then all of them
        const int64_t each = (q + s.tls - 1) / s.tls, lo = s.tl * each, hi = lo + each < q ? lo + each : q;
        Map<VEC> m, before, all; map_clear(m);
        for (int64_t k = lo; k < hi; ++k) if (nv) {
          Map<VEC> t;
          const float *p = work + k * sh.columns + c0, *b = p + sh.chunks * sh.columns;
          load_floats<VEC>(t.P, p, nv); load_floats<VEC>(t.B, b, nv);
          map_behind(t, m); m = t;
        }
        scan_join(s, m, before, all, lds, parity); parity ^= 1;
#pragma unroll
        for (int j = 0; j < VEC; ++j) y[j] = map_at(all.P[j], all.B[j], y[j]);
      }
    }
    for (int64_t k0 = first; k0 < stop; k0 += s.tls) {
      const int64_t k = k0 + s.tl, seg = Op::reverse ? sh.segments - 1 - k : k;
      const bool on = k < stop && nv > 0;
      if (on) op.load(seg);
      float in[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) in[j] = MAPS ? 0.f : y[j];
      if (MAPS || s.tls > 1) {
        Map<VEC> m, before, all;
        map_clear(m);
        if (on) op.map(m);
        scan_join(s, m, before, all, lds, parity); parity ^= 1;
        if (MAPS) { map_behind(all, run); run = all; }
        else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) { in[j] = map_at(before.P[j], before.B[j], y[j]); y[j] = map_at(all.P[j], all.B[j], y[j]); }
        }
      }
      if (!MAPS) {
        if (on) op.run(seg, in);
        if (s.tls == 1) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) y[j] = in[j];
        }
      }
    }
    if (s.tl == 0 && nv) {
      if (MAPS) { store_pack<float, VEC>(work + q * sh.columns + c0, run.P, nv); store_pack<float, VEC>(work + (sh.chunks + q) * sh.columns + c0, run.B, nv); }
      else if (end && stop == sh.segments) store_pack<float, VEC>(end + c0, y, nv);
    }
  }
}
