// learn_recurrence.inl -- the gated recurrence, its gradient, and the advantages, as steps of learn_scan.inl

// the flags of a segment's steps, as they were loaded (a load that is not looked at yet does not have to be waited for); behind the n there are: 0
template <int N> struct Flags {
  uint32_t b[SEG][N];
  __device__ __forceinline__ void load(const uint8_t *flags, int64_t stride, int64_t t0, int n, const int64_t (&row)[N]) {
    if (flags && n == SEG) {      // (apart, so that nothing stands between the loads)
#pragma unroll
      for (int i = 0; i < SEG; ++i) {
#pragma unroll
        for (int j = 0; j < N; ++j) b[i][j] = flags[(t0 + i) * stride + row[j]];
      }
    } else {
#pragma unroll
      for (int i = 0; i < SEG; ++i) {
#pragma unroll
        for (int j = 0; j < N; ++j) { b[i][j] = 0; if (flags && i < n) b[i][j] = flags[(t0 + i) * stride + row[j]]; }
      }
    }
  }
  __device__ __forceinline__ void bits(unsigned (&out)[N]) const {      // bit i: step i
#pragma unroll
    for (int j = 0; j < N; ++j) {
      out[j] = 0;
#pragma unroll
      for (int i = 0; i < SEG; ++i) out[j] |= b[i][j] ? 1u << i : 0u;
    }
  }
};
// the steps of a segment; behind the n there are: `none`
template <class T, int VEC> __device__ __forceinline__ void load_steps(Raw<T, VEC> (&out)[SEG], const Rows<const T> &p, const Place &w, int n, float none) {
  uint32_t off = p.offset(w);
  uintptr_t at = p.first(w);
  if (n == SEG) {
    here(off);
#pragma unroll
    for (int i = 0; i < SEG; ++i, at += p.step()) load_raw<T, VEC>(out[i], device_ptr<const T>(at, off));
  } else {
    here(off);
#pragma unroll
    for (int i = 0; i < SEG; ++i, at += p.step()) {
      if (i < n) load_raw<T, VEC>(out[i], device_ptr<const T>(at, off));
      else out[i].all(from_f<T>(none));
    }
  }
}
__device__ __forceinline__ int steps_left(int64_t steps, const Place &w) { const int64_t t0 = w.base + w.t; return steps - t0 < SEG ? (int)(steps - t0) : SEG; }
static __device__ const float kTiny = 1.17549435e-38f;
// SEG steps of VEC columns; nothing stands between the stores of a whole segment
template <class T, int VEC> __device__ __forceinline__ void write_steps(const Rows<T> &p, const Place &w, int n, const float (&v)[SEG][VEC]) {
  uint32_t off = p.offset(w);
  uintptr_t at = p.first(w);
  if (n == SEG) {
    here(off);
#pragma unroll
    for (int i = 0; i < SEG; ++i, at += p.step()) store_pack<T, VEC>(device_ptr<T>(at, off), v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < SEG; ++i, at += p.step()) if (i < n) store_pack<T, VEC>(device_ptr<T>(at, off), v[i]);
  }
}
// P y + B, where nothing of y passes a P of 0: only an infinite or NaN y has to ask
template <int VEC> __device__ __forceinline__ bool all_finite(const float (&y)[VEC]) {
  bool ok = true;
#pragma unroll
  for (int j = 0; j < VEC; ++j) ok = ok && fabsf(y[j]) < INFINITY;
  return ok;
}
template <int VEC> __device__ __forceinline__ void steps_at(float (&B)[SEG][VEC], const float (&P)[SEG][VEC], const float (&y)[VEC]) {
  if (all_finite<VEC>(y)) {
#pragma unroll
    for (int i = 0; i < SEG; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) B[i][j] = fmaf(P[i][j], y[j], B[i][j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < SEG; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) B[i][j] = map_at(P[i][j], B[i][j], y[j]);
    }
  }
}

// the reset flags of a thread's columns: ROWS = 1 where they always belong to one row (width a multiple of VEC), VEC otherwise
template <int VEC, int ROWS> struct Resets {
  const uint8_t *reset; int64_t rs, width; int64_t row[ROWS];
  __device__ __forceinline__ void place(int64_t c) {
    if (!reset) return;
    // (64-bit division is a hundred instructions, 32-bit a quarter of that)
    const int64_t r = c <= 0x7fffffff && width <= 0x7fffffff ? (int64_t)((uint32_t)c / (uint32_t)width) : c / width;
    int64_t in = c - r * width, at = r;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) { row[j] = at; if (++in == width) { in = 0; ++at; } }
  }
};

__device__ __forceinline__ Place mark_place(const Place &w) { return Place{w.base / SEG, w.cbase, w.t / SEG, w.c}; }      // (base is a multiple of SEG, also below 0)

template <class T, int VEC, int ROWS> struct RecurrenceOp {
  static const bool reverse = false; static const int waves = 4;
  Rows<const T> x, gate; Resets<VEC, ROWS> resets; Rows<T> h; Rows<float> marks; int64_t steps;      // marks: a row for every segment
  Raw<T, VEC> xv[SEG], gv[SEG]; Flags<ROWS> flags; float P[SEG][VEC], B[SEG][VEC];
  __device__ __forceinline__ void start(int64_t c) { resets.place(c); }
  __device__ __forceinline__ void load(const Place &w) {
    const int n = steps_left(steps, w);
    load_steps<T, VEC>(xv, x, w, n, 0.f);
    load_steps<T, VEC>(gv, gate, w, n, INFINITY);      // (a step that is not there keeps the state)
    flags.load(resets.reset, resets.rs, w.base + w.t, n, resets.row);
  }
  __device__ __forceinline__ void prep(Map<VEC> &m) {
    unsigned cut[ROWS]; float least[ROWS];
    flags.bits(cut);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) least[j] = kTiny;
#pragma unroll
    for (int i = 0; i < SEG; ++i) {
      bool c[ROWS];
#pragma unroll
      for (int j = 0; j < ROWS; ++j) { c[j] = (cut[j] >> i) & 1; least[j] = c[j] ? 0.f : least[j]; }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int o = ROWS == 1 ? 0 : j;
        float f, q; sigmoid2(gv[i][j], f, q);
        m.B[j] = fmaf(f, c[o] ? 0.f : m.B[j], q * xv[i][j]);
        m.P[j] = fmaxf(f * (c[o] ? 0.f : m.P[j]), least[o]);
        P[i][j] = m.P[j]; B[i][j] = m.B[j];
      }
    }
  }
  __device__ __forceinline__ void write(const Place &w, const float (&y)[VEC]) {
    if (marks.p) { const Place s = mark_place(w); store_pack<float, VEC>(device_ptr<float>(marks.first(s), marks.offset(s)), y); }
    steps_at<VEC>(B, P, y);
    write_steps<T, VEC>(h, w, steps_left(steps, w), B);
  }
};

// E[t] = what reaches h[t-1] = keep f (dh[t] + E[t+1]); G = dh[t] + E[t+1]; dx = (1 - f) G; dgate = G (p - x) f (1 - f).  p, what a step saw of the state, is
// worked out again from the state kept in front of the segment: in 32 bits, where h itself was rounded, and with fewer bytes than h.  The steps are gone
// through again from dh, 1 - f and w = (p - x) f (1 - f): three quarters of the registers that P and B of every step would take, and with them another wavefront.
template <class T, int VEC, int ROWS> struct RecurrenceGradOp {
  static const bool reverse = true; static const int waves = VEC == 2 ? 3 : 4;      // (pairs: four would spill; 128 x 512 x 64 bf16 16 us with three, 19 with four)
  Rows<const T> x, gate, dh; Resets<VEC, ROWS> resets; Rows<const float> marks; Rows<T> dx, dgate; int64_t steps;
  Raw<T, VEC> xv[SEG], gv[SEG], dn[SEG], dv[SEG]; float mark[VEC]; Flags<ROWS> flags; unsigned cut[ROWS]; float q[SEG][VEC], w[SEG][VEC];
  __device__ __forceinline__ void start(int64_t c) { resets.place(c); }
  __device__ __forceinline__ void load(const Place &w) {
    const int n = steps_left(steps, w);
    load_steps<T, VEC>(xv, x, w, n, 0.f);
    load_steps<T, VEC>(gv, gate, w, n, INFINITY);
    if (dh.p) load_steps<T, VEC>(dn, dh, w, n, 0.f);
    else {
#pragma unroll
      for (int i = 0; i < SEG; ++i) dn[i].all(from_f<T>(0.f));
    }
    const Place s = mark_place(w);
    load_floats<VEC>(mark, device_ptr<const float>(marks.first(s), marks.offset(s)));
    flags.load(resets.reset, resets.rs, w.base + w.t, n, resets.row);
  }
  __device__ __forceinline__ void prep(Map<VEC> &m) {
    float s[VEC], f[SEG][VEC], least[ROWS];
    flags.bits(cut);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) least[j] = kTiny;
#pragma unroll
    for (int j = 0; j < VEC; ++j) s[j] = mark[j];
#pragma unroll
    for (int i = 0; i < SEG; ++i) {
      dv[i] = dn[i];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        sigmoid2(gv[i][j], f[i][j], q[i][j]);
        const float v = xv[i][j], p = (cut[ROWS == 1 ? 0 : j] >> i) & 1 ? 0.f : s[j];
        s[j] = fmaf(f[i][j], p, q[i][j] * v);
        w[i][j] = (p - v) * (f[i][j] * q[i][j]);
      }
    }
#pragma unroll
    for (int i = SEG - 1; i >= 0; --i) {
      bool c[ROWS];
#pragma unroll
      for (int j = 0; j < ROWS; ++j) { c[j] = (cut[j] >> i) & 1; least[j] = c[j] ? 0.f : least[j]; }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const int o = ROWS == 1 ? 0 : j;
        m.B[j] = c[o] ? 0.f : f[i][j] * (dv[i][j] + m.B[j]);
        m.P[j] = fmaxf(f[i][j] * (c[o] ? 0.f : m.P[j]), least[o]);
      }
    }
  }
  __device__ __forceinline__ void write(const Place &at, const float (&y)[VEC]) {
    const int n = steps_left(steps, at);
    float E[VEC], a[SEG][VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) E[j] = y[j];
#pragma unroll
    for (int i = SEG - 1; i >= 0; --i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float G = dv[i][j] + E[j];
        E[j] = (cut[ROWS == 1 ? 0 : j] >> i) & 1 ? 0.f : (1.f - q[i][j]) * G;
        a[i][j] = q[i][j] * G; w[i][j] *= G;
      }
    }
    write_steps<T, VEC>(dx, at, n, a);
    write_steps<T, VEC>(dgate, at, n, w);
  }
};

template <class T, int VEC> struct AdvantageOp {
  static const bool reverse = true; static const int waves = 3;
  Rows<const float> reward; Rows<const T> value, final_value; const T *next_value; const uint8_t *terminated, *truncated; int64_t es, us;
  float gamma, gl; Rows<float> advantage, returns; int64_t steps;
  int64_t row[VEC]; int n; Raw<float, VEC> r[SEG]; Raw<T, VEC> v[SEG], after, f[SEG]; Flags<VEC> term, trunc; float P[SEG][VEC], B[SEG][VEC], V[SEG][VEC];
  __device__ __forceinline__ void start(int64_t c) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) row[j] = c + j;
  }
  __device__ __forceinline__ void load(const Place &w) {
    const int64_t t0 = w.base + w.t;
    n = steps_left(steps, w);
    load_steps<float, VEC>(r, reward, w, n, 0.f);
    load_steps<T, VEC>(v, value, w, n, 0.f);
    load_raw<T, VEC>(after, t0 + n < steps ? device_ptr<const T>(value.first(w) + SEG * value.step(), value.offset(w)) : next_value + row[0]);      // (t0 + n < steps: n = SEG)
    term.load(terminated, es, t0, n, row);
    trunc.load(truncated, us, t0, n, row);
    if (final_value.p) load_steps<T, VEC>(f, final_value, w, n, 0.f);
  }
  __device__ __forceinline__ void prep(Map<VEC> &m) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float then = after[j], least = kTiny;
#pragma unroll
      for (int i = SEG - 1; i >= 0; --i) {
        const bool there = i < n, end = term.b[i][j] != 0, off = !end && trunc.b[i][j] != 0, cut = end || off || (gl == 0.f && there);
        const float now = v[i][j];
        float d = end ? r[i][j] - now : fmaf(gamma, off && final_value.p ? f[i][j] : then, r[i][j]) - now;
        if (off && !final_value.p) d = 0.f;
        least = cut ? 0.f : least;
        const float b = fmaf(gl, cut ? 0.f : m.B[j], d), p = fmaxf(gl * (cut ? 0.f : m.P[j]), least);
        m.B[j] = there ? b : m.B[j]; m.P[j] = there ? p : m.P[j];
        then = there ? now : then;
        P[i][j] = m.P[j]; B[i][j] = m.B[j]; V[i][j] = now;
      }
    }
  }
  __device__ __forceinline__ void write(const Place &w, const float (&y)[VEC]) {
    const int m = steps_left(steps, w);
    steps_at<VEC>(B, P, y);
    write_steps<float, VEC>(advantage, w, m, B);
#pragma unroll
    for (int i = 0; i < SEG; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) B[i][j] += V[i][j];
    }
    write_steps<float, VEC>(returns, w, m, B);
  }
};

template <class Op, int VEC, int MODE>
__global__ __launch_bounds__(256, Op::waves) void k_scan(Op op, const ScanShape sh, const float *start, float *end, float *work) {
  __shared__ ScanLds<VEC> lds;
  scan_columns<Op, VEC, MODE>(op, sh, start, end, work, lds);
}

// one step: elementwise, 8 columns of a row's per thread where rows allow it
template <class T, int VEC>
__global__ __launch_bounds__(256) void k_recurrence_step(const T *__restrict__ x, const T *__restrict__ gate, const float *__restrict__ state, const uint8_t *__restrict__ reset,
    T *__restrict__ h, float *__restrict__ last, float *__restrict__ marks, int64_t columns, int64_t width) {
  for (int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC; c < columns; c += (int64_t)gridDim.x * 256 * VEC) {
    Resets<VEC, 1> at = {reset, 0, width, {0}};
    at.place(c);
    Raw<T, VEC> xv, gv; float s[VEC] = {}, out[VEC];
    load_raw<T, VEC>(xv, x + c); load_raw<T, VEC>(gv, gate + c);
    if (state) load_floats<VEC>(s, state + c);
    const bool cut = reset && reset[at.row[0]];
    if (marks) store_pack<float, VEC>(marks + c, s);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float f, q; sigmoid2(gv[j], f, q);
      out[j] = fmaf(f, cut ? 0.f : s[j], q * xv[j]);
    }
    store_pack<T, VEC>(h + c, out); store_pack<float, VEC>(last + c, out);
  }
}
__global__ __launch_bounds__(256) void k_copy_state(const float *from, float *to, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = from ? from[i] : 0.f;
}

// ---- host: the shape of a launch ---------------------------------------------------------------------------------------------------------------
static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
// 4 bytes of a column row per lane (one f32, two 16-bit columns: 16 bytes took twice the registers and half the wavefronts, and ran at 0.65 of the speed), and
//   column lanes    the most that leave 1024 workgroups (4 per CU), but 16 at least: 64 bytes side by side.  256 x 4096 x 32 f32 with 2^4 .. 2^8 lanes: 109, 97, 88, 82,
//                   103 us; 512 x 64 x 128: 15.9 us with 2^4, 17.8 with 2^3, 21.8 with 2^5.
//   few columns     where that leaves fewer than 512 workgroups, a long rollout (8 turns of a workgroup or more) is cut into chunks of 2^5 lanes for 1024 of them:
//                   2000 x 2048 forward 23.9 us, its gradient 34.7, against 24.9 and 47.4 in one launch of 2^2 or 2^3 lanes; a short one gets 2^3 or 2^2 lanes instead:
//                   advantages of 256 x 4096 8.9 us, against 14.6 in chunks
//   far steps       a thread's 32-bit offset reaches over the workgroup's time lanes: where steps lie so far apart (reach bytes at most) that it could not, one
//                   time lane is left
static ScanShape scan_shape(int64_t steps, int64_t columns, int vec, int64_t reach) {
  ScanShape s;
  s.columns = columns; s.segments = ceil_div(steps, SEG); s.chunks = 1;
  const int64_t lanes = ceil_div(columns, vec);
  const auto groups = [&](int cl) { return ceil_div(lanes, (int64_t)1 << cl); };
  const auto turns = [&](int cl) { return ceil_div(s.segments, 256 >> cl); };
  int most = 8;
  while (most > 0 && ((int64_t)1 << (most - 1)) >= lanes) --most;      // no more column lanes than columns
  int cl = 8;
  while (cl > 4 && groups(cl) < 1024 && (256 >> cl) < s.segments) --cl;
  if (groups(cl) < 512 && turns(cl) >= 8) {
    cl = most < 5 ? most : 5;
    const int64_t want = ceil_div(1024, groups(cl));
    s.chunks = (int)(want < turns(cl) ? want : turns(cl));
  } else {
    while (cl > 2 && groups(cl) < 512 && (256 >> cl) < s.segments) --cl;
    if (cl > most) cl = most;
  }
  if ((256 >> cl) * SEG * reach + 4096 >= ((int64_t)1 << 32)) { cl = 8; s.chunks = 1; }
  s.cl_log = cl; s.groups = groups(cl); s.slots = s.groups < 16 ? s.groups : (s.groups + 7) / 8 * 8;
  s.chunk_segments = ceil_div(turns(cl), s.chunks) * (256 >> cl);
  s.chunks = (int)ceil_div(s.segments, s.chunk_segments);
  return s;
}
static int64_t scan_work(int64_t steps, int64_t columns) {      // floats for any type's launch
  int64_t most = 0;
  if (steps == 0 || columns == 0) return 0;
  for (int vec = 1; vec <= 2; ++vec) { const ScanShape s = scan_shape(steps, columns, vec, 0); if (s.chunks > 1 && 2 * (int64_t)s.chunks * columns > most) most = 2 * (int64_t)s.chunks * columns; }
  return most;
}

template <class Op, int VEC> static void scan_launch(const Op &op, const ScanShape &sh, const float *start, float *end, float *work, hipStream_t st) {
  const unsigned gx = (unsigned)(sh.slots < (1 << 20) ? sh.slots : 1 << 20);
  if (sh.chunks > 1) {
    k_scan<Op, VEC, MAPS><<<dim3(gx, sh.chunks - 1), 256, 0, st>>>(op, sh, start, end, work);
    k_scan<Op, VEC, CHUNK><<<dim3(gx, sh.chunks), 256, 0, st>>>(op, sh, start, end, work);
  } else k_scan<Op, VEC, WHOLE><<<dim3(gx, 1), 256, 0, st>>>(op, sh, start, end, work);
}
