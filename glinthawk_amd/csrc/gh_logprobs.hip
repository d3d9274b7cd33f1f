// Log probabilities of given tokens, the entropy of a row of logits and its largest values.
//
// With m the row's maximum, S = sum e^(x - m) and T = sum e^(x - m) (x - m):
//   ln p(x) = x - m - ln S,   entropy = - sum p ln p = ln S - T / S.
// All three are kept as a pass goes: where the maximum grows by d, S becomes e^-d S and T becomes e^-d (T - d S).
//
// A part of a row is held in the registers of a work-group, so that the logits are read once, all pieces asked for at the start.  The largest values come out of
// them as whole numbers: a value's bits in the order of the values, then its index the other way round, so that no two are equal and the lower index of equal
// values is the larger number.  Every thread knows its own largest; a wave's n-th largest of those is a number that n values at least reach, and so is the
// largest such number of all waves.  What reaches it (mostly a few times n) goes to LDS and is ranked by counting; where that are more than fit, the numbers come
// out one after the other, each the largest below the one before.
// Rows of one part are finished by their work-group.  Longer ones, and few rows, are cut into parts whose S, T, m and sorted largest numbers a second kernel joins.
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

__device__ __forceinline__ void finish_row( const Outputs& o, uint64_t row, Sums z, const uint32_t* tokens, uint32_t vocab, float given )
{
  const float m = z.m == -INFINITY ? 0.0f : z.m;
  const float log_s = logf( z.s );
  if ( o.logprob != nullptr && tokens[row] < vocab ) {
    o.logprob[row] = z.m == -INFINITY ? __builtin_nanf( "" ) : ( given - m ) - log_s;
  }
  if ( o.entropy != nullptr ) {
    o.entropy[row] = log_s - z.t / z.s;
  }
}

// grid: (parts, rows); a part: `per_part` columns, at most THREADS * PIECES * V.  One part: the row is finished here, else parts go to `sums`, `tops`.
template<typename T, int THREADS, int PIECES>
__global__ __launch_bounds__( THREADS ) void logprob_kernel( Outputs o, const T* __restrict__ logits, uint64_t row_stride, const uint32_t* __restrict__ tokens, uint32_t vocab,
                                                            uint32_t n_top, uint32_t per_part, Sums* __restrict__ sums, uint64_t* __restrict__ tops )
{
  constexpr int V = 16 / sizeof( T ), WAVES = THREADS / WAVE;
  struct Piece
  {
    T e[V];
  };
  __shared__ Sums s_sums[WAVES];
  __shared__ uint64_t s_reach[WAVES];
  __shared__ uint64_t s_number[CANDIDATES];
  __shared__ uint32_t s_count;
  const uint32_t wave = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
  const uint64_t row = blockIdx.y;
  const T* x = logits + row * row_stride;
  const uint32_t c0 = blockIdx.x * per_part, n = min( vocab - c0, per_part );

  Piece piece[PIECES];
#pragma unroll
  for ( int p = 0; p < PIECES; p++ ) {
    const uint32_t i = ( p * THREADS + threadIdx.x ) * V;
    if ( i + V <= n ) {
      __builtin_memcpy( &piece[p], x + c0 + i, 16 ); // rows may begin anywhere
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

  Sums z { -INFINITY, 0.0f, 0.0f };
  uint32_t best_i = 0;
#pragma unroll
  for ( int p = 0; p < PIECES; p++ ) {
#pragma unroll
    for ( int e = 0; e < V; e++ ) {
      const float v = to_f32( piece[p].e[e] );
      best_i = v > z.m ? ( p * THREADS + threadIdx.x ) * V + e : best_i; // the first of equal ones, as indices rise
      z.m = fmaxf( z.m, v );
    }
  }
  const float m = z.m == -INFINITY ? 0.0f : z.m;
  float s4[4] = { 0, 0, 0, 0 }, t4[4] = { 0, 0, 0, 0 };
#pragma unroll
  for ( int p = 0; p < PIECES; p++ ) {
#pragma unroll
    for ( int e = 0; e < V; e++ ) {
      const float d = to_f32( piece[p].e[e] ) - m, w = __builtin_amdgcn_exp2f( d * LOG2E );
      s4[e & 3] += w;
      t4[e & 3] = __builtin_fmaf( w, fmaxf( d, -1e30f ), t4[e & 3] ); // (a weight of 0 times -inf counts nothing)
    }
  }
  z.s = ( s4[0] + s4[1] ) + ( s4[2] + s4[3] );
  z.t = ( t4[0] + t4[1] ) + ( t4[2] + t4[3] );
  const uint64_t mine = z.m == -INFINITY ? 0 : number_of( z.m, best_i );
#pragma unroll
  for ( int off = 1; off < WAVE; off <<= 1 ) {
    z = join( z, Sums { __shfl_xor( z.m, off, WAVE ), __shfl_xor( z.s, off, WAVE ), __shfl_xor( z.t, off, WAVE ) } );
  }
  uint64_t reach = 0;
  if ( n_top != 0 ) {
    uint32_t rank = 0; // lanes of the wave with a larger number (or an equal one, no value, and a lower lane)
#pragma unroll 4
    for ( uint32_t i = 0; i < WAVE; i++ ) {
      const uint64_t other = (uint64_t)__builtin_amdgcn_readlane( (int)( mine >> 32 ), i ) << 32 | (uint32_t)__builtin_amdgcn_readlane( (int)(uint32_t)mine, i );
      rank += other > mine || ( other == mine && i < lane );
    }
    const uint64_t which = __builtin_amdgcn_ballot_w64( rank == n_top - 1 );
    const int at = __builtin_ctzll( which );
    reach = (uint64_t)__builtin_amdgcn_readlane( (int)( mine >> 32 ), at ) << 32 | (uint32_t)__builtin_amdgcn_readlane( (int)(uint32_t)mine, at );
  }
  if ( lane == 0 ) {
    s_sums[wave] = z;
    s_reach[wave] = reach;
  }
  __syncthreads();
  z = s_sums[0];
  reach = s_reach[0];
  for ( int w = 1; w < WAVES; w++ ) {
    z = join( z, s_sums[w] );
    reach = max( reach, s_reach[w] );
  }
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
  const float max_m = z.m == -INFINITY ? 0.0f : z.m, log_s = logf( z.s );
  auto put = [&]( uint32_t rank, uint64_t number ) {
    if ( gridDim.x != 1 ) {
      tops[part * n_top + rank] = number == 0 ? 0 : ( number & 0xffffffff00000000ull ) | (uint32_t)~( index_of( number ) + c0 );
    } else {
      o.top_ids[row * n_top + rank] = index_of( number );
      o.top_logprobs[row * n_top + rank] = ( value_of( number ) - max_m ) - log_s;
    }
  };
  const float reach_value = value_of( reach );
#pragma unroll
  for ( int p = 0; p < PIECES; p++ ) {
#pragma unroll
    for ( int e = 0; e < V; e++ ) {
      const float v = to_f32( piece[p].e[e] );
      if ( !( v < reach_value ) ) { // few come this far
        const uint32_t i = ( p * THREADS + threadIdx.x ) * V + e;
        const uint64_t number = number_of( v, i );
        if ( i < n && number >= reach ) {
          const uint32_t at = atomicAdd( &s_count, 1u ); // (their order does not matter: each is ranked among all)
          if ( at < CANDIDATES ) {
            s_number[at] = number;
          }
        }
      }
    }
  }
  __syncthreads();
  const uint32_t count = s_count;
  if ( count <= CANDIDATES ) {
    for ( uint32_t i = threadIdx.x; i < count; i += THREADS ) {
      const uint64_t number = s_number[i];
      uint32_t rank = 0;
      for ( uint32_t k = 0; k < count; k++ ) {
        rank += s_number[k] > number;
      }
      if ( rank < n_top ) {
        put( rank, number );
      }
    }
    for ( uint32_t i = count + threadIdx.x; i < n_top; i += THREADS ) { // a part of fewer columns than alternatives
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

// columns of a piece differ with the type; the workspace has to serve every type, so the parts are those of fp32 pieces of four
LogprobPlan plan_logprobs( uint64_t rows, uint64_t vocab, uint32_t n_top )
{
  LogprobPlan p {};
  constexpr uint64_t MOST = 32768; // columns of a part at most
  const uint64_t wanted = std::max<uint64_t>( 1, (uint64_t)cu_count() / std::max<uint64_t>( rows, 1 ) );  // few rows: a part for every CU
  uint64_t parts = std::max<uint64_t>( ( vocab + MOST - 1 ) / MOST, std::min<uint64_t>( wanted, std::min<uint64_t>( vocab / 4096, 16 ) ) );
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
    go( many, std::integral_constant<int, 4> {} );
  } else {
    go( many, std::integral_constant<int, 8> {} );
  }
}

} // namespace
} // namespace gh

using namespace gh;

extern "C" {

uint64_t gh_token_logprobs_workspace( uint64_t rows, uint64_t vocab, uint32_t n_top ) { return rows == 0 || vocab == 0 ? 0 : plan_logprobs( rows, vocab, n_top ).bytes; }

int gh_token_logprobs( float* logprob, float* entropy, uint32_t* top_ids, float* top_logprobs, const void* logits, uint64_t row_stride, const uint32_t* tokens_dev,
                       uint64_t vocab, uint64_t rows, uint32_t n_top, gh_dtype dt, void* workspace, uint64_t workspace_bytes, gh_stream stream )
{
  if ( rows != 0 ) { // what can be said without a device is said first
    GH_REQUIRE( logits && ( logprob == nullptr || tokens_dev ) && ( n_top == 0 || ( top_ids && top_logprobs ) ), "gh_token_logprobs: NULL pointer" );
    GH_REQUIRE( dt == GH_F16 || dt == GH_F32 || dt == GH_BF16, "gh_token_logprobs: unsupported dtype %d", (int)dt );
    GH_REQUIRE( vocab > 0 && vocab <= 1u << 21 && rows <= 65535, "gh_token_logprobs: bad shape (up to 65535 rows of up to 2097152 values)" );
    GH_REQUIRE( n_top <= MAX_TOP && n_top <= vocab, "gh_token_logprobs: %u alternatives of %llu values (at most %u)", n_top, (unsigned long long)vocab, MAX_TOP );
    GH_REQUIRE( row_stride >= vocab || rows == 1, "gh_token_logprobs: rows of %llu values lie %llu apart", (unsigned long long)vocab, (unsigned long long)row_stride );
    GH_REQUIRE( reinterpret_cast<uintptr_t>( logits ) % dtype_size( dt ) == 0, "gh_token_logprobs: logits are not aligned to their elements" );
  }
  if ( int rc = ensure_init() ) {
    return rc;
  }
  if ( rows == 0 ) {
    return GH_OK;
  }
  const LogprobPlan p = plan_logprobs( rows, vocab, n_top );
  GH_REQUIRE( p.bytes == 0 || ( workspace != nullptr && reinterpret_cast<uintptr_t>( workspace ) % 16 == 0 ), "gh_token_logprobs: a 16-byte aligned workspace is needed" );
  if ( p.bytes > workspace_bytes ) {
    return fail( GH_ERR_WORKSPACE, "gh_token_logprobs: workspace of %llu bytes, %llu are needed", (unsigned long long)workspace_bytes, (unsigned long long)p.bytes );
  }
  uint64_t* tops = static_cast<uint64_t*>( workspace );
  Sums* sums = reinterpret_cast<Sums*>( tops + rows * p.parts * n_top );
  const Outputs o { logprob, entropy, top_ids, top_logprobs };
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

} // extern "C"
