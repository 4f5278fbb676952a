// learn_recurrence.inl -- the gated recurrence, its gradient, and the advantages, as steps of learn_scan.inl

static const int SEG = AGARCL_MARK_STEPS;

// flags of a segment: bit i of out[j] for step i and column j.  Rows of a step are the columns / width.
template <int VEC> __device__ __forceinline__ void load_flags(unsigned (&out)[VEC], const uint8_t *flags, int64_t stride, int64_t t0, int n, const int64_t (&row)[VEC], bool one_row, int nv) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) out[j] = 0;
  if (!flags) return;
  if (one_row) {
    unsigned bits = 0;
#pragma unroll
    for (int i = 0; i < SEG; ++i) if (i < n) bits |= flags[(t0 + i) * stride + row[0]] ? 1u << i : 0u;
#pragma unroll
    for (int j = 0; j < VEC; ++j) out[j] = bits;
  } else {
#pragma unroll
    for (int i = 0; i < SEG; ++i) if (i < n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) if (j < nv) out[j] |= flags[(t0 + i) * stride + row[j]] ? 1u << i : 0u;
    }
  }
}

template <class T, int VEC> __device__ __forceinline__ void load_steps(Raw<T, VEC> (&out)[SEG], const T *p, int64_t stride, int n, int nv) {
  if (n == SEG && nv == VEC) {      // (apart, so that nothing stands between the loads)
#pragma unroll
    for (int i = 0; i < SEG; ++i) load_raw<T, VEC>(out[i], p + i * stride, VEC);
  } else {
#pragma unroll
    for (int i = 0; i < SEG; ++i) load_raw<T, VEC>(out[i], p + i * stride, i < n ? nv : 0);
  }
}
template <class T, int VEC> __device__ __forceinline__ void anew(Raw<T, VEC> (&r)[SEG]) {
#pragma unroll
  for (int i = 0; i < SEG; ++i) r[i].anew();
}

template <class T, int VEC> struct RecurrenceOp {
  static const bool reverse = false;
  const T *x, *gate; int64_t xs, gs; const uint8_t *reset; int64_t rs; T *h; float *marks; int64_t steps, columns, width;
  int64_t c0, row[VEC]; int nv, n; Raw<T, VEC> xv[SEG], gv[SEG]; unsigned cut[VEC];
  __device__ __forceinline__ void place(int64_t c, int m) {
    c0 = c; nv = m;
#pragma unroll
    for (int j = 0; j < VEC; ++j) row[j] = reset ? (c + j) / width : 0;
  }
  __device__ __forceinline__ void load(int64_t seg) {
    const int64_t t0 = seg * SEG;
    n = steps - t0 < SEG ? (int)(steps - t0) : SEG;
    load_steps<T, VEC>(xv, x + t0 * xs + c0, xs, n, nv);
    load_steps<T, VEC>(gv, gate + t0 * gs + c0, gs, n, nv);
    load_flags<VEC>(cut, reset, rs, t0, n, row, width % VEC == 0, nv);
  }
  __device__ __forceinline__ void step(int i, int j, float &y, float &f) const {
    float q; sigmoid2(gv[i][j], f, q);
    y = fmaf(f, (cut[j] >> i) & 1 ? 0.f : y, q * xv[i][j]);
  }
  __device__ __forceinline__ void map(Map<VEC> &m) const {
#pragma unroll
    for (int i = 0; i < SEG; ++i) if (i < n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) { float f; step(i, j, m.B[j], f); m.P[j] = (cut[j] >> i) & 1 ? 0.f : map_p(m.P[j], fmaxf(f, 1.17549435e-38f)); }
    }
  }
  __device__ __forceinline__ void run(int64_t seg, float (&y)[VEC]) {
    const int64_t t0 = seg * SEG;
    anew(gv);
    if (marks) store_pack<float, VEC>(marks + seg * columns + c0, y, nv);
#pragma unroll
    for (int i = 0; i < SEG; ++i) if (i < n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) { float f; step(i, j, y[j], f); }
      store_pack<T, VEC>(h + (t0 + i) * columns + c0, y, nv);
    }
  }
};

// E[t] = what reaches h[t-1] = keep f (dh[t] + E[t+1]); G = dh[t] + E[t+1]; dx = (1 - f) G; dgate = G (p - x) f (1 - f).  p, what a step saw of the state, is
// worked out again from the state kept in front of the segment: in 32 bits, where h itself was rounded, and with fewer bytes than h.
template <class T, int VEC> struct RecurrenceGradOp {
  static const bool reverse = true;
  const T *x, *gate, *dh; int64_t xs, gs, ds; const uint8_t *reset; int64_t rs; const float *marks; T *dx, *dgate; int64_t steps, columns, width;
  int64_t c0, row[VEC]; int nv, n; Raw<T, VEC> xv[SEG], gv[SEG], dv[SEG]; unsigned cut[VEC]; float mark[VEC];
  __device__ __forceinline__ void place(int64_t c, int m) {
    c0 = c; nv = m;
#pragma unroll
    for (int j = 0; j < VEC; ++j) row[j] = reset ? (c + j) / width : 0;
  }
  __device__ __forceinline__ void load(int64_t seg) {
    const int64_t t0 = seg * SEG;
    n = steps - t0 < SEG ? (int)(steps - t0) : SEG;
    load_steps<T, VEC>(xv, x + t0 * xs + c0, xs, n, nv);
    load_steps<T, VEC>(gv, gate + t0 * gs + c0, gs, n, nv);
    if (dh) load_steps<T, VEC>(dv, dh + t0 * ds + c0, ds, n, nv);
    else {
#pragma unroll
      for (int i = 0; i < SEG; ++i) dv[i] = Raw<T, VEC>{};
    }
    load_floats<VEC>(mark, marks + seg * columns + c0, nv);
    load_flags<VEC>(cut, reset, rs, t0, n, row, width % VEC == 0, nv);
  }
  __device__ __forceinline__ void map(Map<VEC> &m) const {
#pragma unroll
    for (int i = SEG - 1; i >= 0; --i) if (i < n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float f, q; sigmoid2(gv[i][j], f, q);
        const bool c = (cut[j] >> i) & 1;
        m.B[j] = c ? 0.f : f * (dv[i][j] + m.B[j]);
        m.P[j] = c ? 0.f : map_p(m.P[j], fmaxf(f, 1.17549435e-38f));
      }
    }
  }
  __device__ __forceinline__ void run(int64_t seg, float (&y)[VEC]) {
    const int64_t t0 = seg * SEG;
    anew(gv);
    float p[SEG][VEC], s[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[j] = mark[j];
#pragma unroll
    for (int i = 0; i < SEG; ++i) if (i < n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float f, q; sigmoid2(gv[i][j], f, q);
        p[i][j] = (cut[j] >> i) & 1 ? 0.f : s[j];
        s[j] = fmaf(f, p[i][j], q * xv[i][j]);
      }
    }
    anew(gv);
#pragma unroll
    for (int i = SEG - 1; i >= 0; --i) if (i < n) {
      float a[VEC], b[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float f, q; sigmoid2(gv[i][j], f, q);
        const float G = dv[i][j] + y[j];
        a[j] = q * G; b[j] = G * (p[i][j] - xv[i][j]) * f * q;
        y[j] = (cut[j] >> i) & 1 ? 0.f : f * G;
      }
      store_pack<T, VEC>(dx + (t0 + i) * columns + c0, a, nv);
      store_pack<T, VEC>(dgate + (t0 + i) * columns + c0, b, nv);
    }
  }
};

template <class T, int VEC> struct AdvantageOp {
  static const bool reverse = true;
  const float *reward; const T *value, *next_value; const uint8_t *terminated, *truncated; const T *final_value; int64_t rs, vs, es, us, fs;
  float gamma, gl; float *advantage, *returns; int64_t steps, columns;
  int64_t c0, row[VEC]; int nv, n; Raw<float, VEC> r[SEG]; Raw<T, VEC> v[SEG], after, fv[SEG]; unsigned term[VEC], trunc[VEC];
  __device__ __forceinline__ void place(int64_t c, int m) {
    c0 = c; nv = m;
#pragma unroll
    for (int j = 0; j < VEC; ++j) row[j] = c + j;
  }
  __device__ __forceinline__ void load(int64_t seg) {
    const int64_t t0 = seg * SEG;
    n = steps - t0 < SEG ? (int)(steps - t0) : SEG;
    load_steps<float, VEC>(r, reward + t0 * rs + c0, rs, n, nv);
    load_steps<T, VEC>(v, value + t0 * vs + c0, vs, n, nv);
    load_raw<T, VEC>(after, t0 + n < steps ? value + (t0 + n) * vs + c0 : next_value + c0, nv);
    load_flags<VEC>(term, terminated, es, t0, n, row, false, nv);
    load_flags<VEC>(trunc, truncated, us, t0, n, row, false, nv);
    if (final_value) load_steps<T, VEC>(fv, final_value + t0 * fs + c0, fs, n, nv);
  }
  __device__ __forceinline__ void step(int i, int j, float &A, bool &cut) const {
    const float now = v[i][j], then = i + 1 < n ? v[i + 1 < SEG ? i + 1 : i][j] : after[j];
    const bool end = (term[j] >> i) & 1, off = !end && (trunc[j] >> i) & 1;
    cut = end || off;
    float d = end ? r[i][j] - now : fmaf(gamma, off && final_value ? fv[i][j] : then, r[i][j]) - now;
    if (off && !final_value) d = 0.f;
    A = cut || gl == 0.f ? d : fmaf(gl, A, d);
  }
  __device__ __forceinline__ void map(Map<VEC> &m) const {
#pragma unroll
    for (int i = SEG - 1; i >= 0; --i) if (i < n) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) { bool cut; step(i, j, m.B[j], cut); m.P[j] = cut ? 0.f : map_p(m.P[j], gl); }
    }
  }
  __device__ __forceinline__ void run(int64_t seg, float (&A)[VEC]) const {
    const int64_t t0 = seg * SEG;
#pragma unroll
    for (int i = SEG - 1; i >= 0; --i) if (i < n) {
      float ret[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) { bool cut; step(i, j, A[j], cut); ret[j] = A[j] + v[i][j]; }
      store_pack<float, VEC>(advantage + (t0 + i) * columns + c0, A, nv);
      store_pack<float, VEC>(returns + (t0 + i) * columns + c0, ret, nv);
    }
  }
};

template <class Op, int VEC, bool MAPS>
__global__ __launch_bounds__(256) void k_scan(Op op, const ScanShape sh, const float *start, float *end, float *work) {
  __shared__ ScanLds<VEC> lds;
  scan_columns<Op, VEC, MAPS>(op, sh, start, end, work, lds);
}

__global__ __launch_bounds__(256) void k_copy_state(const float *from, float *to, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = from ? from[i] : 0.f;
}

// ---- host: the shape of a launch ---------------------------------------------------------------------------------------------------------------
static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
struct ScanPlan { int vec; ScanShape sh; };
static ScanPlan scan_plan(int64_t steps, int64_t columns, int wide) {
  ScanPlan p; ScanShape &s = p.sh;
  s.columns = columns; s.segments = ceil_div(steps, SEG); if (s.segments < 1) s.segments = 1;
  p.vec = ceil_div(columns, wide) * s.segments >= 32768 ? wide : 1;
  const int64_t lanes = ceil_div(columns, p.vec);
  const int least = p.vec == 4 ? 2 : p.vec == 2 ? 3 : 4;                       // 64 bytes of f32 side by side
  int cl = 8;
  while (cl > 0 && ((int64_t)1 << (cl - 1)) >= lanes) --cl;    // no more column lanes than columns
  while (cl > least && ceil_div(lanes, (int64_t)1 << cl) < 1024 && (256 >> cl) < s.segments) --cl;
  s.cl_log = cl;
  s.groups = ceil_div(lanes, (int64_t)1 << cl);
  const int64_t tls = 256 >> cl, rounds = ceil_div(s.segments, tls);
  s.chunks = 1;
  if (s.groups < 512 && rounds >= 4) { const int64_t want = ceil_div(1024, s.groups); s.chunks = (int)(want < rounds ? want : rounds); if (s.chunks > 256) s.chunks = 256; }
  s.chunk_segments = ceil_div(ceil_div(s.segments, s.chunks), tls) * tls;
  s.chunks = (int)ceil_div(s.segments, s.chunk_segments);
  return p;
}
static int64_t scan_work(int64_t steps, int64_t columns) {      // enough for either width
  int64_t most = 0;
  for (int wide = 2; wide <= 4; wide += 2) { const ScanPlan p = scan_plan(steps, columns, wide); if (p.sh.chunks > 1 && 2 * (int64_t)p.sh.chunks * columns > most) most = 2 * (int64_t)p.sh.chunks * columns; }
  return most;
}

template <class Op, int VEC> static void scan_launch(const Op &op, const ScanShape &sh, const float *start, float *end, float *work, hipStream_t st) {
  const unsigned gx = (unsigned)(sh.groups < (1 << 20) ? sh.groups : 1 << 20);
  if (sh.chunks > 1) k_scan<Op, VEC, true><<<dim3(gx, sh.chunks - 1), 256, 0, st>>>(op, sh, start, end, work);
  k_scan<Op, VEC, false><<<dim3(gx, sh.chunks), 256, 0, st>>>(op, sh, start, end, work);
}
