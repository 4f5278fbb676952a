// learn_recurrence.inl -- the gated recurrence, its gradient, and the advantages, as steps of learn_scan.inl

// the flags of a segment's steps, as they were loaded (a load that is not looked at yet does not have to be waited for)
template <int N> struct Flags {
  uint32_t b[SEG][N];
  __device__ __forceinline__ void load(const Rows<const uint8_t> &p, const Place &w, const uint32_t (&c)[N]) {      // c: in place of w.c
    uintptr_t at = p.first(w);
    const uint32_t off = w.t * (uint32_t)p.stride;
#pragma unroll
    for (int i = 0; i < SEG; ++i, at += p.step()) {
      const auto r = span(at, p.p);
#pragma unroll
      for (int j = 0; j < N; ++j) b[i][j] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, if_there(off + c[j], i < w.n), 0, 0);
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
// the steps of a segment; 0 behind those that there are
template <class T, int VEC> __device__ __forceinline__ void load_steps(Raw<T, VEC> (&out)[SEG], const Rows<const T> &p, const Place &w) {
  const uint32_t off = p.offset(w);
  uintptr_t at = p.first(w);
#pragma unroll
  for (int i = 0; i < SEG; ++i, at += p.step()) fetch<T, VEC>(out[i], span(at, p.p), if_there(off, i < w.n));
}
static __device__ const float kTiny = 1.17549435e-38f;
template <class T, int VEC> __device__ __forceinline__ void write_steps(const Rows<T> &p, const Place &w, const float (&v)[SEG][VEC]) {
  const uint32_t off = p.offset(w);
  uintptr_t at = p.first(w);
#pragma unroll
  for (int i = 0; i < SEG; ++i, at += p.step()) put<T, VEC>(span(at, p.p), if_there(off, i < w.n), v[i]);
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

// (64-bit division is a hundred instructions, 32-bit a quarter of that)
__device__ __forceinline__ int64_t row_of(int64_t c, int64_t width) { return c <= 0x7fffffff && width <= 0x7fffffff ? (int64_t)((uint32_t)c / (uint32_t)width) : c / width; }
// the reset flags of a thread's columns: ROWS = 1 where they always belong to one row (width a multiple of VEC), VEC otherwise
template <int VEC, int ROWS> struct Resets {
  Rows<const uint8_t> reset; int64_t width; int64_t base; uint32_t row[ROWS];      // the rows behind row `base`, that of the workgroup's first column
  __device__ __forceinline__ void place(int64_t cbase, int64_t c) {
    base = 0;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) row[j] = 0;
    if (!reset.p) return;
    base = row_of(cbase, width);
    const int64_t r = row_of(c, width);
    int64_t in = c - r * width, at = r - base;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) { row[j] = (uint32_t)at; if (++in == width) { in = 0; ++at; } }
  }
  __device__ __forceinline__ void load(Flags<ROWS> &f, const Place &w) const { f.load(reset, Place{w.base, base, w.t, 0, w.n}, row); }
};

__device__ __forceinline__ Place mark_place(const Place &w) { return Place{w.base / SEG, w.cbase, w.t / SEG, w.c, w.n}; }

// a step that is not there keeps the state
template <class T, int VEC> __device__ __forceinline__ void keep_behind(Raw<T, VEC> (&gate)[SEG], int n) {
  if (n == SEG) return;
#pragma unroll
  for (int i = 0; i < SEG; ++i) if (i >= n) gate[i].all(from_f<T>(INFINITY));
}

// The memory: P = f P, B = f B + (1 - f) x, one exp and one reciprocal per element for both f and 1 - f.  HBM bounds it where there are columns enough: 256 x 4096 x 64
// bf16 with the marks 89 us (4.9 TB/s), x 32 f32 82 us (5.1 TB/s); a large copy runs at 4.76 TB/s.  Few columns: 20000 x 4 x 64 f32 28 us in two launches, each at 3.7
// TB/s of what it moves, x and gate twice.
template <class T, int VEC, int ROWS> struct RecurrenceOp {
  static const bool reverse = false; static const int waves = 4;
  Rows<const T> x, gate; Resets<VEC, ROWS> resets; Rows<T> h; Rows<float> marks;      // marks: a row for every segment
  Raw<T, VEC> xv[SEG], gv[SEG]; Flags<ROWS> flags; int n; float P[SEG][VEC], B[SEG][VEC];
  __device__ __forceinline__ void start(int64_t cbase, int64_t c) { resets.place(cbase, c); }
  __device__ __forceinline__ void load(const Place &w) {
    n = w.n;
    load_steps<T, VEC>(xv, x, w);
    load_steps<T, VEC>(gv, gate, w);
    resets.load(flags, w);
  }
  __device__ __forceinline__ void prep(Map<VEC> &m) {
    unsigned cut[ROWS]; float least[ROWS];
    flags.bits(cut);
    keep_behind<T, VEC>(gv, n);
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
    const Place s = mark_place(w);
    put<float, VEC>(span(marks.first(s), marks.p), if_there(marks.offset(s), w.n > 0), y);
    steps_at<VEC>(B, P, y);
    write_steps<T, VEC>(h, w, B);
  }
};

// E[t] = what reaches h[t-1] = keep f (dh[t] + E[t+1]); G = dh[t] + E[t+1]; dx = (1 - f) G; dgate = G (p - x) f (1 - f).  p, what a step saw of the state, is
// worked out again from the state kept in front of the segment: in 32 bits, where h itself was rounded, and with fewer bytes than h.  The steps are gone
// through again from dh, the lesser of f and 1 - f (sigmoid_again makes both of it) and w = (p - x) f (1 - f): three quarters of the registers that P and B of every step
// would take, and with them another wavefront.
// Bound by HBM as the forward pass is: 256 x 4096 x 64 bf16 147 us (4.8 TB/s), x 32 f32 138 us (5.0); 20000 x 4 x 64 f32 41 us in two launches.
template <class T, int VEC, int ROWS> struct RecurrenceGradOp {
  static const bool reverse = true; static const int waves = VEC == 2 ? 3 : 4;      // (pairs: with the registers of four, half of the types spill)
  Rows<const T> x, gate, dh; Resets<VEC, ROWS> resets; Rows<const float> marks; Rows<T> dx, dgate;
  Raw<T, VEC> xv[SEG], gv[SEG], dn[SEG], dv[SEG]; Raw<float, VEC> mark; int n; Flags<ROWS> flags; unsigned cut[ROWS]; float s[SEG][VEC], w[SEG][VEC];
  __device__ __forceinline__ void start(int64_t cbase, int64_t c) { resets.place(cbase, c); }
  __device__ __forceinline__ void load(const Place &w) {
    n = w.n;
    load_steps<T, VEC>(xv, x, w);
    load_steps<T, VEC>(gv, gate, w);
    load_steps<T, VEC>(dn, dh, w);
    const Place s = mark_place(w);
    fetch<float, VEC>(mark, span(marks.first(s), marks.p), if_there(marks.offset(s), w.n > 0));
    resets.load(flags, w);
  }
  __device__ __forceinline__ void prep(Map<VEC> &m) {
    float h[VEC], f[SEG][VEC], least[ROWS];
    flags.bits(cut);
    keep_behind<T, VEC>(gv, n);
#pragma unroll
    for (int j = 0; j < ROWS; ++j) least[j] = kTiny;
#pragma unroll
    for (int j = 0; j < VEC; ++j) h[j] = mark[j];
#pragma unroll
    for (int i = 0; i < SEG; ++i) {
      dv[i] = dn[i];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float q; s[i][j] = sigmoid2(gv[i][j], f[i][j], q);
        const float v = xv[i][j], p = (cut[ROWS == 1 ? 0 : j] >> i) & 1 ? 0.f : h[j];
        h[j] = fmaf(f[i][j], p, q * v);
        w[i][j] = (p - v) * (f[i][j] * q);
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
    float E[VEC], a[SEG][VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) E[j] = y[j];
#pragma unroll
    for (int i = SEG - 1; i >= 0; --i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float G = dv[i][j] + E[j];
        float f, q; sigmoid_again(s[i][j], f, q);
        E[j] = (cut[ROWS == 1 ? 0 : j] >> i) & 1 ? 0.f : f * G;
        a[i][j] = q * G; w[i][j] *= G;
      }
    }
    write_steps<T, VEC>(dx, at, a);
    write_steps<T, VEC>(dgate, at, w);
  }
};

// The advantages: P = gamma lambda, or 0 where an episode ends, B = delta + gamma lambda B.  22 bytes per element; a rollout of usual size is one turn, and that turn's
// latency (loads, three joins, stores) is all its time: 256 x 4096 9 us, 32 x 64 5; 30001 x 5 in two launches 6 + 8.
template <class T, int VEC> struct AdvantageOp {
  static const bool reverse = true; static const int waves = 4;
  Rows<const float> reward; Rows<const T> value, next_value, final_value; Rows<const uint8_t> terminated, truncated;
  float gamma, gl; Rows<float> advantage, returns; int64_t steps;
  int n; bool last; Raw<float, VEC> r[SEG]; Raw<T, VEC> v[SEG], after, behind, f[SEG]; Flags<VEC> terminated_, truncated_; float P[SEG][VEC], B[SEG][VEC], V[SEG][VEC];
  __device__ __forceinline__ void start(int64_t, int64_t) { }
  __device__ __forceinline__ void load(const Place &w) {
    n = w.n; last = w.base + w.t + n >= steps;
    uint32_t c[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) c[j] = w.c + j;
    load_steps<float, VEC>(r, reward, w);
    load_steps<T, VEC>(v, value, w);
    fetch<T, VEC>(after, span(value.first(w) + SEG * value.step(), true), if_there(value.offset(w), n && !last));
    fetch<T, VEC>(behind, span(next_value.first(Place{0, w.cbase, 0, w.c, n}), true), if_there(w.c * (uint32_t)sizeof(T), n && last));
    terminated_.load(terminated, w, c);
    truncated_.load(truncated, w, c);
    load_steps<T, VEC>(f, final_value, w);
  }
  __device__ __forceinline__ void prep(Map<VEC> &m) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float then = last ? behind[j] : after[j], least = kTiny;
#pragma unroll
      for (int i = SEG - 1; i >= 0; --i) {
        const bool there = i < n, end = terminated_.b[i][j] != 0, off = !end && truncated_.b[i][j] != 0, cut = end || off || (gl == 0.f && there);
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
    steps_at<VEC>(B, P, y);
    write_steps<float, VEC>(advantage, w, B);
#pragma unroll
    for (int i = 0; i < SEG; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) B[i][j] += V[i][j];
    }
    write_steps<float, VEC>(returns, w, B);
  }
};

template <class Op, int VEC, int MODE>
__global__ __launch_bounds__(256, Op::waves) void k_scan(Op op, const ScanShape sh, const float *start, float *end, float *work) {
  __shared__ ScanLds<VEC> lds;
  scan_columns<Op, VEC, MODE>(op, sh, start, end, work, lds);
}

// One step: elementwise, 4 columns of a row's per thread where rows allow it.  4096 x 256 bf16 (14.7 MB) 3.7 us on the GPU, 4 TB/s; a launch alone takes 3.4 in a row of launches.
template <class T, int VEC>
__global__ __launch_bounds__(256) void k_recurrence_step(const T *__restrict__ x, const T *__restrict__ gate, const float *__restrict__ state, const uint8_t *__restrict__ reset,
    T *__restrict__ h, float *__restrict__ last, float *__restrict__ marks, int64_t columns, int64_t width) {
  for (int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC; c < columns; c += (int64_t)gridDim.x * 256 * VEC) {
    Raw<T, VEC> xv, gv; float s[VEC] = {}, out[VEC];
    load_raw<T, VEC>(xv, x + c); load_raw<T, VEC>(gv, gate + c);
    if (state) load_floats<VEC>(s, state + c);
    const bool cut = reset && reset[row_of(c, width)];
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
//   column lanes    2^8, where that leaves 512 workgroups (2 per CU): one time lane, nothing to join.  256 x 4096 x 64 bf16 forward and gradient 89 and 147 us, with 2^7
//                   97 and 157.  Otherwise the most that leave 640: 256 x 3000 x 64 bf16 with 2^8 .. 2^5 lanes 77, 70, 73, 77 us and 127, 114, 120, 122; 64 x 1024 x 64
//                   with 2^7 .. 2^4 12.6, 10.8, 10.2, 13.8 and 17.8, 15.7, 14.7, 19.9.  16 at least: 64 bytes side by side
//   few columns     2^3, where 2^4 lanes leave fewer than 256 workgroups, or fewer than 512 of a short rollout: 500 x 2560 f32 with 2^4, 2^3, 2^2 11.7, 10.5, 11.7 us
//                   (gradient 15.4, 14.8, 16.0), 500 x 4096 12.7, 11.7, 14.6; 1500 x 4096 31.8, 34.4, 45.4.  2^2, where 2^3 leave fewer than 150: 900 x 1024 9.9,
//                   with 2^3 12.7.  2^0, where 2^2 leave 16 or fewer: 900 x 64 6.5, with 2^2 7.4
//   chunks          of a long rollout of few columns, for 1280 workgroups: 1500 x 2560 f32 21.4 us, 23.7 without, gradient 29.2 and 44; 900 x 2560 16.8 and 16.4, 21.1 and
//                   22.9; 900 x 256 9.6 and 7.6; 2500 x 64 10 and 10.6, gradient 11.4 and 19.6; 1500 x 64 9.9 and 7.7; 5000 x 4096 97 and 95, 131 and 138.  2^6 lanes, but
//                   2^5 where there would be so many chunks that the joining of their maps takes long: 20000 x 256 27.8 us, 30.5 with 2^6; 4000 x 2048 44 and 41
//   far steps       a thread's 32-bit offset reaches over the workgroup's time lanes: where steps lie so far apart (reach bytes at most) that it could not, one
//                   time lane is left
static ScanShape scan_shape(int64_t steps, int64_t columns, int vec, int64_t reach) {
  ScanShape s;
  s.columns = columns; s.steps = steps; s.segments = ceil_div(steps, SEG); s.chunks = 1;
  const int64_t lanes = ceil_div(columns, vec);
  const auto groups = [&](int cl) { return ceil_div(lanes, (int64_t)1 << cl); };
  const auto turns = [&](int cl) { return ceil_div(s.segments, 256 >> cl); };
  int most = 8;
  while (most > 0 && ((int64_t)1 << (most - 1)) >= lanes) --most;      // no more column lanes than columns
  int cl = 8;
  while (cl > 4 && groups(cl) < (cl == 8 ? 512 : 640) && (256 >> cl) < s.segments) --cl;
  if (cl == 4 && s.segments > 16) {
    const int64_t n = groups(4);
    if (n < 256 || (n < 512 && s.segments <= 64)) cl = 3;
    if (groups(3) < 150 && s.segments > 32) cl = 2;
    if (groups(2) <= 16 && s.segments > 64) cl = 0;
    if (n < 256 && s.segments > (cl == 0 ? 256 : 128)) {
      cl = groups(6) >= 16 ? 6 : 5;
      if (cl > most) cl = most;
      const int64_t want = ceil_div(1280, groups(cl));
      s.chunks = (int)(want < turns(cl) ? want : turns(cl));
    }
  }
  if (cl > most) cl = most;
  if ((256 >> cl) * SEG * reach + 4096 >= ((int64_t)1 << 31)) { cl = 8; s.chunks = 1; }
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
