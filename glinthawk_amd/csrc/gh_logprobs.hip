// Log probabilities of given tokens, the entropy of a row of logits and its largest values.
//
// With m the row's maximum, S = sum e^(x - m) and T = sum e^(x - m) (x - m):
//   ln p(x) = x - m - ln S,   entropy = - sum p ln p = ln S - T / S.
// All three are kept as a pass goes: where the maximum grows by d, S becomes e^-d S and T becomes e^-d (T - d S).
//
// A part of a row is held in the registers of a work-group, so that the logits are read once, all pieces asked for at the start: bound by the bytes for many rows (and
// nearly by the vector ALU: some 12 slots a value), by latency for few.  2047 rows of 32000 f16 values, 20 alternatives: 41 us (3.2 TB/s), without alternatives 27 (4.9);
// 7 rows in fp32, 5 alternatives: 7.7 us.  Sums made piece by piece as the loads land, each thread relative to its own maximum, were no faster (43 us): the
// work-groups of a CU are in different phases already.
// The largest values: of the threads' own largest, each wave finds one that q of its threads reach and few more; half the waves have q threads that reach the middle one of
// those, so with q = 2 n / waves at least n values do, and of many thousand only some more.  They go to LDS as whole numbers, a value's bits in the order of the values, then its index the other way
// round, so that no two are equal and the lower index of equal values is the larger number, and are ranked by counting.  Where they are more than fit since many are equal
// (a row that lets few tokens through is -inf elsewhere), the row is read again for what is larger and for as many of the equal ones as are wanted: 2047 rows of which
// 30 of 32000 f16 values are finite, 20 alternatives, 102 us a call on its own (50 with all of them finite).  Where even what is larger is more than fit (a row whose
// values are in order), the numbers come out one after the other, each the largest below the one before (2047 such rows, 20 alternatives: 1030 us).
// Rows of one part are finished by their work-group.  Longer ones are cut into parts whose S, T, m and sorted largest numbers a second kernel joins.
#include "gh_common.h"

#include <algorithm>

namespace gh {
namespace {

constexpr uint32_t MAX_TOP = 64, MAX_PARTS = 64;
constexpr uint32_t CANDIDATES = 1024;
constexpr float LOG2E = 1.4426950408889634f;

struct Outputs
{
  float* logprob;
  float* entropy;
  uint32_t* top_ids;
  float* top_logprobs;
  bool fills; // logprob of a token that is none: `fill`, or left as it is
  float fill;
};

// ---- numbers in the order of the values --------------------------------------------------------
__device__ __forceinline__ uint64_t number_of( float v, uint32_t index )
{
  const uint32_t bits = __builtin_bit_cast( uint32_t, v + 0.0f ); // (-0 is 0)
  const uint32_t order = v != v ? 0u : bits >> 31 ? ~bits : bits | 0x80000000u;
  return (uint64_t)order << 32 | (uint32_t)~index;
}
__device__ __forceinline__ uint32_t index_of( uint64_t number ) { return ~(uint32_t)number; }
__device__ __forceinline__ float value_of( uint64_t number )
{
  const uint32_t order = (uint32_t)( number >> 32 );
  return __builtin_bit_cast( float, order == 0 ? 0x7fc00000u : order >> 31 ? order & 0x7fffffffu : ~order );
}

__device__ __forceinline__ uint64_t wave_max_u64( uint64_t v )
{
#pragma unroll
  for ( int off = 32; off > 0; off >>= 1 ) {
    v = max( v, (uint64_t)__shfl_xor( (unsigned long long)v, off, WAVE ) );
  }
  return v;
}

// A value that at least k of a wave's lanes reach, and few more than k: of distances from the largest, the k-th by its upper 16 bits, then the farthest lane within it.
// (64 alternatives of 2047 rows: 50 us; with one maximum after the other 60.)
// v without NaN, k at most 64, largest: of the wave.
__device__ __forceinline__ float reached_by( float v, float largest, uint32_t k )
{
  if ( k == 1 ) {
    return largest;
  }
  const uint32_t d = v == largest ? 0u : __builtin_bit_cast( uint32_t, largest - v );
  uint32_t within = 0x7fffffffu;
#pragma unroll
  for ( int bit = 30; bit >= 16; bit-- ) {
    const uint32_t less = within - ( 1u << bit );
    within = (uint32_t)__popcll( __builtin_amdgcn_ballot_w64( d <= less ) ) >= k ? less : within;
  }
  return -wave_max( d <= within ? -v : -INFINITY );
}

// 16 bytes of a row
template<typename T>
struct RowPiece
{
  static constexpr int V = 16 / sizeof( T );
  union
  {
    uint4 raw;
    T e[V];
  };
  // Each pass over the registers makes fp32 values of its own: kept from one to the next they would take twice the registers of the pieces.
  __device__ __forceinline__ void forget() { asm volatile( "" : "+v"( raw.x ), "+v"( raw.y ), "+v"( raw.z ), "+v"( raw.w ) ); }
  __device__ __forceinline__ float best() const // without NaN
  {
    if constexpr ( std::is_same_v<T, __half> ) { // two at a time
      typedef _Float16 f16x2 __attribute__( ( ext_vector_type( 2 ) ) );
      const f16x2 a = __builtin_elementwise_max( __builtin_bit_cast( f16x2, raw.x ), __builtin_bit_cast( f16x2, raw.y ) );
      const f16x2 b = __builtin_elementwise_max( __builtin_bit_cast( f16x2, raw.z ), __builtin_bit_cast( f16x2, raw.w ) );
      const f16x2 c = __builtin_elementwise_max( a, b );
      return fmaxf( fmaxf( -INFINITY, (float)c.x ), (float)c.y );
    } else {
      float b = -INFINITY;
#pragma unroll
      for ( int k = 0; k < V; k++ ) {
        b = fmaxf( b, to_f32( e[k] ) );
      }
      return b;
    }
  }
};

struct Sums
{
  float m, s, t;
};
// S and T of two parts, relative to the larger maximum; a part that has seen -inf only weighs nothing
__device__ __forceinline__ Sums join( Sums a, Sums b )
{
  Sums r;
  r.m = fmaxf( a.m, b.m );
  const float m = r.m == -INFINITY ? 0.0f : r.m;
  const float da = fmaxf( a.m - m, -1e30f ), db = fmaxf( b.m - m, -1e30f );
  const float wa = __builtin_amdgcn_exp2f( da * LOG2E ), wb = __builtin_amdgcn_exp2f( db * LOG2E );
  r.s = wa * a.s + wb * b.s;
  r.t = wa * __builtin_fmaf( da, a.s, a.t ) + wb * __builtin_fmaf( db, b.s, b.t );
  return r;
}

// S and T from sums over 2^d and 2^d d with d = x log2(e) - c: c is m log2(e) but for its rounding, which is taken out here.  The largest value's own weight is what
// the sum is divided by, so that S is 1 at least (no log probability above 0), and T is no more than 0 (no entropy below 0).
__device__ __forceinline__ Sums sums_of( float max_m, float m, float c, float s, float t )
{
  const float off = __builtin_fmaf( m, LOG2E, -c ); // x log2(e) - c = (x - m) log2(e) + off
  const float w = __builtin_amdgcn_exp2f( off ), below = __builtin_fmaf( -off, s, t );
  return { max_m, s / w, ( below > 0.0f ? 0.0f : below ) / w * 0.693147180559945309417f };
}

__device__ __forceinline__ void finish_row( const Outputs& o, uint64_t row, Sums z, const uint32_t* tokens, uint32_t vocab, float given )
{
  const float m = z.m == -INFINITY ? 0.0f : z.m;
  const float log_s = logf( z.s );
  if ( o.logprob != nullptr ) {
    if ( tokens[row] < vocab ) {
      o.logprob[row] = z.m == -INFINITY ? __builtin_nanf( "" ) : ( given - m ) - log_s;
    } else if ( o.fills ) {
      o.logprob[row] = o.fill;
    }
  }
  if ( o.entropy != nullptr ) {
    o.entropy[row] = log_s - z.t / z.s;
  }
}

// grid: (parts, rows); a part: `per_part` columns, at most THREADS * PIECES * V.  One part: the row is finished here, else parts go to `sums`, `tops`.
template<typename T, int THREADS, int PIECES>
__global__ __launch_bounds__( THREADS, THREADS == 512 || ( THREADS == 1024 && PIECES * 16 / sizeof( T ) <= 32 ) ? 8 : 4 ) void logprob_kernel( Outputs o, const T* __restrict__ logits, uint64_t row_stride, const uint32_t* __restrict__ tokens, uint32_t vocab,
                                                            uint32_t n_top, uint32_t per_part, Sums* __restrict__ sums, uint64_t* __restrict__ tops )
{
  constexpr int V = 16 / sizeof( T ), WAVES = THREADS / WAVE;
  using Piece = RowPiece<T>;
  __shared__ float2 s_sums[WAVES];
  __shared__ float s_best[WAVES], s_reach[WAVES];
  __shared__ uint64_t s_number[CANDIDATES];
  __shared__ uint32_t s_count, s_found[WAVES];
  const uint32_t wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  const uint64_t row = blockIdx.y;
  const T* x = logits + row * row_stride;
  const uint32_t c0 = blockIdx.x * per_part, n = min( vocab - c0, per_part );

  Piece piece[PIECES];
#pragma unroll
  for ( int p = 0; p < PIECES; p++ ) {
    const uint32_t i = ( p * THREADS + threadIdx.x ) * V;
    if ( i + V <= n ) { // rows may begin anywhere
      __builtin_memcpy( &piece[p].raw, x + c0 + i, 16 );
    } else {
#pragma unroll
      for ( int e = 0; e < V; e++ ) {
        piece[p].e[e] = i + e < n ? x[c0 + i + e] : from_f32<T>( -INFINITY );
      }
    }
  }
  float given = 0.0f;
  if ( threadIdx.x == 0 && gridDim.x == 1 && o.logprob != nullptr && tokens[row] < vocab ) {
    given = to_f32( x[tokens[row]] );
  }
  if ( threadIdx.x == 0 ) {
    s_count = 0;
  }

  float best = -INFINITY, piece_best[PIECES];
#pragma unroll
  for ( int p = 0; p < PIECES; p++ ) {
    piece_best[p] = piece[p].best();
    piece[p].forget();
    best = fmaxf( best, piece_best[p] );
  }
  const float wave_best = wave_max( best );
  const float wave_reach = n_top == 0 ? 0.0f : reached_by( best, wave_best, ( n_top + WAVES / 2 - 1 ) / ( WAVES / 2 ) );
  if ( lane == 0 ) {
    s_best[wave] = wave_best;
    s_reach[wave] = wave_reach;
  }
  __syncthreads();
  const float max_m = wave_max( lane < WAVES ? s_best[lane] : -INFINITY ), m = max_m == -INFINITY ? 0.0f : max_m, c = m * LOG2E;
  // f16: in powers of 2, relative to 2^c (see `sums_of`); larger types' values may lie so far from 0 that c's rounding is a large number
  constexpr bool SMALL = std::is_same_v<T, __half>;
  float s4[4] = { 0, 0, 0, 0 }, t4[4] = { 0, 0, 0, 0 };
#pragma unroll
  for ( int p = 0; p < PIECES; p++ ) {
#pragma unroll
    for ( int e = 0; e < V; e++ ) {
      float d, w;
      if constexpr ( SMALL ) {
        d = __builtin_fmaf( to_f32( piece[p].e[e] ), LOG2E, -c ); // one rounding, f16 taken as it is
        w = __builtin_amdgcn_exp2f( d );
      } else {
        d = to_f32( piece[p].e[e] ) - m; // exact where it matters
        w = __builtin_amdgcn_exp2f( d * LOG2E );
      }
      s4[e & 3] += w;
      t4[e & 3] = __builtin_fmaf( w, fmaxf( d, -1e30f ), t4[e & 3] ); // (a weight of 0 times -inf counts nothing)
    }
    piece[p].forget();
  }
  const float wave_s = wave_sum( ( s4[0] + s4[1] ) + ( s4[2] + s4[3] ) ), wave_t = wave_sum( ( t4[0] + t4[1] ) + ( t4[2] + t4[3] ) );
  if ( lane == 0 ) {
    s_sums[wave] = make_float2( wave_s, wave_t );
  }
  float reach = 0.0f;
  if ( n_top != 0 ) {
    // the middle one of the waves' values: as many are larger, or equal and in front
    const float mine = s_reach[lane % WAVES];
    uint32_t rank = 0;
#pragma unroll
    for ( uint32_t w = 0; w < WAVES; w++ ) {
      const float other = lane_value( mine, (int)w );
      rank += other > mine || ( other == mine && w < lane );
    }
    reach = lane_value( mine, __builtin_ctzll( __builtin_amdgcn_ballot_w64( rank == WAVES / 2 - 1 ) ) );
    uint32_t thread = threadIdx.x;
    asm volatile( "" : "+v"( thread ) ); // (the columns' numbers are made here and not ahead of time)
    if ( !( best < reach ) ) { // few threads come this far
#pragma unroll
      for ( int p = 0; p < PIECES; p++ ) {
        if ( !( piece_best[p] < reach ) ) {
#pragma unroll
          for ( int e = 0; e < V; e++ ) {
            const float v = to_f32( piece[p].e[e] );
            const uint32_t i = ( p * THREADS + thread ) * V + e;
            if ( !( v < reach ) && i < n ) { // (NaN comes along: where there is nothing else it is wanted)
              const uint32_t at = atomicAdd( &s_count, 1u ); // (their order does not matter: each is ranked among all)
              if ( at < CANDIDATES ) {
                s_number[at] = number_of( v, i );
              }
            }
          }
        }
      }
    }
  }
  __syncthreads();
  const uint32_t count = s_count;
  if ( count <= CANDIDATES && threadIdx.x >= max( max( count, n_top ), 1u ) ) {
    return; // nothing to rank or to write, and no use for the row's sums
  }
  float2 total = s_sums[0];
#pragma unroll
  for ( int w = 1; w < WAVES; w++ ) {
    total.x += s_sums[w].x;
    total.y += s_sums[w].y;
  }
  const Sums z = SMALL ? sums_of( max_m, m, c, total.x, total.y ) : Sums { max_m, total.x, total.y };
  const uint64_t part = row * gridDim.x + blockIdx.x;
  if ( threadIdx.x == 0 ) {
    if ( gridDim.x == 1 ) {
      finish_row( o, row, z, tokens, vocab, given );
    } else {
      sums[part] = z;
    }
  }
  if ( n_top == 0 ) {
    return;
  }
  const float log_s = logf( z.s );
  auto put = [&]( uint32_t rank, uint64_t number ) {
    if ( gridDim.x != 1 ) {
      tops[part * n_top + rank] = number == 0 ? 0 : ( number & 0xffffffff00000000ull ) | (uint32_t)~( index_of( number ) + c0 );
    } else {
      o.top_ids[row * n_top + rank] = index_of( number );
      o.top_logprobs[row * n_top + rank] = ( value_of( number ) - m ) - log_s;
    }
  };
  uint32_t listed = count;
  if ( count > CANDIDATES ) {
    // More than fit, since many are equal to what is reached (a row that lets few tokens through is -inf elsewhere): the row once more, for what is larger, and then, in the order
    // of their columns and no further than they are wanted, for what is equal; behind -inf for NaN.
    __syncthreads();
    if ( threadIdx.x == 0 ) {
      s_count = 0;
    }
    __syncthreads();
    for ( uint32_t i = threadIdx.x; i < n; i += THREADS ) {
      const float v = to_f32( x[c0 + i] );
      if ( v > reach ) {
        const uint32_t at = atomicAdd( &s_count, 1u );
        if ( at < CANDIDATES ) {
          s_number[at] = number_of( v, i );
        }
      }
    }
    __syncthreads();
    listed = s_count;
    for ( uint32_t look = 0; look < ( reach == -INFINITY ? 2u : 1u ) && listed < n_top; look++ ) {
      for ( uint32_t i0 = 0; i0 < n && listed < n_top; i0 += THREADS ) {
        const uint32_t i = i0 + threadIdx.x;
        const float v = i < n ? to_f32( x[c0 + i] ) : 0.0f;
        const uint64_t have = __builtin_amdgcn_ballot_w64( i < n && ( look == 0 ? v == reach : v != v ) );
        if ( lane == 0 ) {
          s_found[wave] = __popcll( have );
        }
        __syncthreads();
        uint32_t at = listed + __popcll( have & ( ( 1ull << lane ) - 1 ) );
        for ( uint32_t w = 0; w < WAVES; w++ ) {
          at += w < wave ? s_found[w] : 0;
          listed += s_found[w];
        }
        if ( ( have >> lane & 1 ) && at < n_top ) {
          s_number[at] = number_of( v, i );
        }
        __syncthreads();
      }
    }
    listed = s_count >= n_top ? s_count : min( listed, n_top ); // (of the equal ones no more than are wanted were put down)
  }
  if ( listed <= CANDIDATES ) {
    for ( uint32_t i = threadIdx.x; i < listed; i += THREADS ) {
      const uint64_t number = s_number[i];
      uint32_t rank = 0;
#pragma unroll 8
      for ( uint32_t k = 0; k < listed; k++ ) {
        rank += s_number[k] > number;
      }
      if ( rank < n_top ) {
        put( rank, number );
      }
    }
    for ( uint32_t i = listed + threadIdx.x; i < n_top; i += THREADS ) { // a part of fewer columns than alternatives
      put( i, 0 );
    }
    return;
  }
  uint64_t below = ~0ull;
  for ( uint32_t rank = 0; rank < n_top; rank++ ) {
    uint64_t largest = 0;
    for ( uint32_t i = threadIdx.x; i < n; i += THREADS ) {
      const uint64_t number = number_of( to_f32( x[c0 + i] ), i );
      largest = number < below ? max( largest, number ) : largest;
    }
    largest = wave_max_u64( largest );
    __syncthreads();
    if ( lane == 0 ) {
      s_number[wave] = largest;
    }
    __syncthreads();
    for ( int w = 0; w < WAVES; w++ ) {
      largest = max( largest, s_number[w] );
    }
    below = largest;
    if ( threadIdx.x == 0 ) {
      put( rank, largest );
    }
  }
}

// parts of a row joined: one work-group a row.  The parts' numbers are sorted: one's rank is its place plus how many of each other part are larger, found by bisection.
__global__ __launch_bounds__( 256 ) void logprob_join_kernel( Outputs o, const uint32_t* __restrict__ tokens, uint32_t vocab, uint32_t n_top, uint32_t parts,
                                                             const Sums* __restrict__ sums, const uint64_t* __restrict__ tops, const void* __restrict__ logits,
                                                             uint64_t row_stride, int dt )
{
  __shared__ uint64_t s_number[MAX_PARTS * MAX_TOP];
  const uint64_t row = blockIdx.x;
  const uint32_t n = parts * n_top;
  for ( uint32_t i = threadIdx.x; i < n; i += 256 ) {
    s_number[i] = tops[row * n + i];
  }
  Sums z = sums[row * parts];
  for ( uint32_t p = 1; p < parts; p++ ) {
    z = join( z, sums[row * parts + p] );
  }
  if ( threadIdx.x == 0 ) {
    float given = 0.0f;
    if ( o.logprob != nullptr && tokens[row] < vocab ) {
      const uint64_t at = row * row_stride + tokens[row];
      given = dt == GH_F16 ? to_f32( static_cast<const __half*>( logits )[at] )
                           : dt == GH_BF16 ? to_f32( static_cast<const __bf16*>( logits )[at] ) : static_cast<const float*>( logits )[at];
    }
    finish_row( o, row, z, tokens, vocab, given );
  }
  __syncthreads();
  const float m = z.m == -INFINITY ? 0.0f : z.m, log_s = logf( z.s );
  for ( uint32_t i = threadIdx.x; i < n; i += 256 ) {
    const uint64_t number = s_number[i];
    if ( number == 0 ) {
      continue;
    }
    uint32_t rank = 0;
    for ( uint32_t p = 0; p < parts; p++ ) {
      uint32_t low = 0, high = n_top; // how many of the part are larger
      while ( low < high ) {
        const uint32_t middle = ( low + high ) / 2;
        if ( s_number[p * n_top + middle] > number ) {
          low = middle + 1;
        } else {
          high = middle;
        }
      }
      rank += low;
    }
    if ( rank < n_top ) {
      o.top_ids[row * n_top + rank] = index_of( number );
      o.top_logprobs[row * n_top + rank] = ( value_of( number ) - m ) - log_s;
    }
  }
}

struct LogprobPlan
{
  uint32_t threads, pieces, parts, per_part; // per_part: columns
  uint64_t bytes;
};

// A row is one part while it fits the registers of a work-group: more parts for few rows take the launch that joins them, which costs what they save (1 row of 32000
// fp32 values, 5 alternatives: one part 10.8 us, 7 parts and the join 10.4; 64 alternatives 15 and 20).
LogprobPlan plan_logprobs( uint64_t rows, uint64_t vocab, uint32_t n_top )
{
  LogprobPlan p {};
  constexpr uint64_t MOST = 32768; // columns of a part at most
  const uint64_t parts = ( vocab + MOST - 1 ) / MOST;
  p.per_part = (uint32_t)( ( ( vocab + parts - 1 ) / parts + 7 ) / 8 * 8 );
  p.parts = (uint32_t)( ( vocab + p.per_part - 1 ) / p.per_part );
  p.bytes = p.parts == 1 ? 0 : rows * p.parts * ( ( n_top + 2 ) * sizeof( uint64_t ) );
  return p;
}

template<typename T>
void launch_logprobs( const LogprobPlan& p, const Outputs& o, const void* logits, uint64_t row_stride, const uint32_t* tokens, uint32_t vocab, uint64_t rows,
                      uint32_t n_top, Sums* sums, uint64_t* tops, hipStream_t st )
{
  constexpr uint32_t V = 16 / sizeof( T );
  auto go = [&]( auto threads, auto pieces ) {
    constexpr int N = decltype( threads )::value, P = decltype( pieces )::value;
    logprob_kernel<T, N, P><<<dim3( p.parts, (unsigned)rows ), N, 0, st>>>( o, static_cast<const T*>( logits ), row_stride, tokens, vocab, n_top, p.per_part, sums, tops );
  };
  const std::integral_constant<int, 256> few {};
  const std::integral_constant<int, 1024> many {};
  const uint32_t pieces = ( p.per_part + V - 1 ) / V;
  if ( pieces <= 256 ) {
    go( few, std::integral_constant<int, 1> {} );
  } else if ( pieces <= 1024 ) {
    go( few, std::integral_constant<int, 4> {} );
  } else if ( pieces <= 2048 ) {
    go( many, std::integral_constant<int, 2> {} );
  } else if ( pieces <= 4096 ) {
    // f16: more work-groups a CU, whose short phases fill each other's gaps (rows of 32000, 20 alternatives, calls with 512 and with 1024 threads, us: 384 rows 14.3 and 14.5, 448
    // 14.6 and 15.2, 768 19.7 and 21.7, 2047 38.3 and 44.9, 4096 62.6 and 80.8; up to 320 equal.  256 threads, 2047 rows: 43.  bf16 does not fit the registers so: 47 and 47)
    if constexpr ( std::is_same_v<T, __half> ) {
      if ( rows >= 512 ) {
        go( std::integral_constant<int, 512> {}, std::integral_constant<int, 8> {} );
        return;
      }
    }
    go( many, std::integral_constant<int, 4> {} );
  } else if constexpr ( sizeof( T ) == 4 ) { // (a part has up to 32768 columns)
    go( many, std::integral_constant<int, 8> {} );
  }
}

// Both entry points
int token_logprobs( const char* op, const Outputs& o, const void* logits, uint64_t row_stride, const uint32_t* tokens_dev, uint64_t vocab, uint64_t rows, uint32_t n_top,
                    gh_dtype dt, void* workspace, uint64_t workspace_bytes, gh_stream stream )
{
  if ( rows != 0 ) { // what can be said without a device is said first
    GH_REQUIRE( logits && ( o.logprob == nullptr || tokens_dev ) && ( n_top == 0 || ( o.top_ids && o.top_logprobs ) ), "%s: NULL pointer", op );
    GH_REQUIRE( dt == GH_F16 || dt == GH_F32 || dt == GH_BF16, "%s: unsupported dtype %d", op, (int)dt );
    GH_REQUIRE( vocab > 0 && vocab <= 1u << 21 && rows <= 65535, "%s: bad shape (up to 65535 rows of up to 2097152 values)", op );
    GH_REQUIRE( n_top <= MAX_TOP && n_top <= vocab, "%s: %u alternatives of %llu values (at most %u)", op, n_top, (unsigned long long)vocab, MAX_TOP );
    GH_REQUIRE( row_stride >= vocab || rows == 1, "%s: rows of %llu values lie %llu apart", op, (unsigned long long)vocab, (unsigned long long)row_stride );
    GH_REQUIRE( reinterpret_cast<uintptr_t>( logits ) % dtype_size( dt ) == 0, "%s: logits are not aligned to their elements", op );
  }
  if ( int rc = ensure_init() ) {
    return rc;
  }
  if ( rows == 0 ) {
    return GH_OK;
  }
  const LogprobPlan p = plan_logprobs( rows, vocab, n_top );
  GH_REQUIRE( p.bytes == 0 || ( workspace != nullptr && reinterpret_cast<uintptr_t>( workspace ) % 16 == 0 ), "%s: a 16-byte aligned workspace is needed", op );
  if ( p.bytes > workspace_bytes ) {
    return fail( GH_ERR_WORKSPACE, "%s: workspace of %llu bytes, %llu are needed", op, (unsigned long long)workspace_bytes, (unsigned long long)p.bytes );
  }
  uint64_t* tops = static_cast<uint64_t*>( workspace );
  Sums* sums = reinterpret_cast<Sums*>( tops + rows * p.parts * n_top );
  hipStream_t st = as_stream( stream );
  switch ( dt ) {
    case GH_F16: launch_logprobs<__half>( p, o, logits, row_stride, tokens_dev, (uint32_t)vocab, rows, n_top, sums, tops, st ); break;
    case GH_BF16: launch_logprobs<__bf16>( p, o, logits, row_stride, tokens_dev, (uint32_t)vocab, rows, n_top, sums, tops, st ); break;
    default: launch_logprobs<float>( p, o, logits, row_stride, tokens_dev, (uint32_t)vocab, rows, n_top, sums, tops, st ); break;
  }
  GH_LAUNCH_CHECK();
  if ( p.parts > 1 ) {
    logprob_join_kernel<<<(unsigned)rows, 256, 0, st>>>( o, tokens_dev, (uint32_t)vocab, n_top, p.parts, sums, tops, logits, row_stride, (int)dt );
    GH_LAUNCH_CHECK();
  }
  return GH_OK;
}

} // namespace
} // namespace gh

using namespace gh;

extern "C" {

uint64_t gh_token_logprobs_workspace( uint64_t rows, uint64_t vocab, uint32_t n_top ) { return rows == 0 || vocab == 0 ? 0 : plan_logprobs( rows, vocab, n_top ).bytes; }

int gh_token_logprobs( float* logprob, float* entropy, uint32_t* top_ids, float* top_logprobs, const void* logits, uint64_t row_stride, const uint32_t* tokens_dev,
                       uint64_t vocab, uint64_t rows, uint32_t n_top, gh_dtype dt, void* workspace, uint64_t workspace_bytes, gh_stream stream )
{
  return token_logprobs( "gh_token_logprobs", { logprob, entropy, top_ids, top_logprobs, false, 0.0f }, logits, row_stride, tokens_dev, vocab, rows, n_top, dt, workspace, workspace_bytes, stream );
}

int gh_token_logprobs_fill( float* logprob, float fill, float* entropy, uint32_t* top_ids, float* top_logprobs, const void* logits, uint64_t row_stride,
                            const uint32_t* tokens_dev, uint64_t vocab, uint64_t rows, uint32_t n_top, gh_dtype dt, void* workspace, uint64_t workspace_bytes, gh_stream stream )
{
  return token_logprobs( "gh_token_logprobs_fill", { logprob, entropy, top_ids, top_logprobs, true, fill }, logits, row_stride, tokens_dev, vocab, rows, n_top, dt, workspace, workspace_bytes, stream );
}

} // extern "C"
