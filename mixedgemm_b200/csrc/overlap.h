// Host side: do the buffers of a call share memory?  Exact, also for rows that lie between the rows of another
// buffer (columns of one tensor), and without a loop over rows unless pitches differ and the buffers interleave.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <initializer_list>

namespace mg {

// `rows` runs of `bytes`, `pitch` bytes apart (pitch >= bytes where there are two or more).
struct Span {
  uintptr_t p, end;  // an empty one is (0, 0), which meets nothing
  size_t rows, bytes, pitch;
  Span(const void* ptr, size_t rows_, size_t bytes_, size_t pitch_) : p(0), end(0), rows(rows_), bytes(bytes_), pitch(pitch_) {
    if (!ptr || !rows || !bytes) return;
    p = reinterpret_cast<uintptr_t>(ptr);
    end = p + (rows - 1) * pitch + bytes;
  }
  Span(const void* ptr, size_t bytes_) : Span(ptr, 1, bytes_, bytes_) {}
};

// Does [lo, hi) meet one of `rows` runs of `bytes` at first, first + pitch, ...?
inline bool meets(__int128 lo, __int128 hi, __int128 first, size_t rows, size_t bytes, size_t pitch) {
  const __int128 r = lo < first + (__int128)bytes ? 0 : (lo - first - (__int128)bytes) / (__int128)pitch + 1;
  return r < (__int128)rows && first + r * (__int128)pitch < hi;
}

inline bool rows_overlap(const Span& a, const Span& b) {
  const __int128 a0 = a.p, b0 = b.p;
  if (a.rows == 1) return meets(a0, a0 + a.bytes, b0, b.rows, b.bytes, b.pitch);
  if (b.rows == 1) return meets(b0, b0 + b.bytes, a0, a.rows, a.bytes, a.pitch);
  // one pitch: row r of a and row s of b lie to one another as row 0 of a and row s - r of b
  if (a.pitch == b.pitch)
    return meets(a0, a0 + a.bytes, b0 - (__int128)(a.rows - 1) * a.pitch, a.rows + b.rows - 1, b.bytes, b.pitch);
  const Span &few = a.rows < b.rows ? a : b, &many = a.rows < b.rows ? b : a;
  for (size_t r = 0; r < few.rows; ++r) {
    const __int128 lo = (__int128)few.p + (__int128)r * few.pitch;
    if (meets(lo, lo + few.bytes, many.p, many.rows, many.bytes, many.pitch)) return true;
  }
  return false;
}

inline bool overlap(const Span& a, const Span& b) { return a.p < b.end && b.p < a.end && rows_overlap(a, b); }

// The same rows: what one thread reads from the one it alone writes to the other.
inline bool same(const Span& a, const Span& b) {
  return a.p == b.p && a.rows == b.rows && a.bytes == b.bytes && (a.rows <= 1 || a.pitch == b.pitch);
}

// Does an output share memory with an input or with another output?
inline bool any_overlap(std::initializer_list<Span> outs, std::initializer_list<Span> ins) {
  for (const Span* o = outs.begin(); o != outs.end(); ++o) {
    for (const Span& i : ins)
      if (overlap(*o, i)) return true;
    for (const Span* q = o + 1; q != outs.end(); ++q)
      if (overlap(*o, *q)) return true;
  }
  return false;
}

}  // namespace mg
