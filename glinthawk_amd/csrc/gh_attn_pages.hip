// Attention over a cache in pages: of one new token of every context (decode), and causal attention of packed prompts.
//
// For query row r of context i and head h, with j running over the keys the row attends and row(i, j) the cache row that the page table gives:
//   out = sum_j w_j V[row(i, j)] / sum_j w_j,  w_j = 2^( s_j - m ),  s_j = q . K[row(i, j)] * log2(e) / sqrt(head size),  m the largest s_j so far:
// one pass over the keys, sums and maxima in fp32, what was summed is rescaled where the maximum grows.
// The columns of a (context, kv head) pair are its query rows times the gqa heads that share the kv head, token by token; work-groups take blocks of columns.
// Where there are few work-groups the keys are cut into splits of `chunk`, each of which leaves (sum_j w_j V, m, sum_j w_j) in the workspace for pages_merge_kernel.
#include "gh_pages.h"

#include <algorithm>

namespace gh {
namespace {

constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp2( float x ) { return __builtin_amdgcn_exp2f( x ); }

// What a call's kernels are given: decode has `lengths`, packed prompts `seqs`.
struct Call
{
  Pages pages;
  Packed seqs;
  const uint32_t* lengths;
  uint32_t n_kv_heads, gqa, size;
  uint32_t max_keys; // keys beyond are not attended: what the grid and the partial results are sized for
  uint32_t chunk, splits;
  uint32_t n_blocks; // blocks of columns there may be (decode: of a context)
  uint32_t longest_first; // decode of up to 64 contexts: see block_of
  float scale_log2e;
  float* part_out; // [row][head][split][size]
  float* part_ml;  // [row][head][split][2]
};

// A work-group's share: columns [col0, ...) of sequence seq, whose token 0 is query row row0 and attends keys [0, start + 1)
struct Block
{
  uint32_t seq, h, split, row0, tokens, start, col0;
};

// DECODE: a sequence is a context's one token.  False: nothing to do (for the whole work-group).
template<bool DECODE, uint32_t COLS>
__device__ __forceinline__ bool block_of( const Call& a, uint32_t number, uint32_t h, uint32_t split, Block* b )
{
  b->h = h;
  b->split = split;
  if constexpr ( DECODE ) {
    uint32_t seq = number / a.n_blocks, length;
    b->col0 = number % a.n_blocks * COLS;
    if ( a.longest_first ) { // the context with `seq` longer ones, so that a launch does not end on a long one
      const uint32_t lane = threadIdx.x & 63, mine = lane < a.seqs.batch ? min( a.lengths[lane], a.max_keys ) : 0;
      const uint32_t key = min( mine, 0x3ffffffu ) * 64 + 63 - lane; // no two alike
      uint32_t rank = 0;
#pragma unroll
      for ( int i = 0; i < 64; i++ ) {
        rank += (uint32_t)__builtin_amdgcn_readlane( (int)key, i ) > key ? 1 : 0;
      }
      seq = (uint32_t)__builtin_ctzll( __builtin_amdgcn_ballot_w64( rank == seq ) );
      length = (uint32_t)__builtin_amdgcn_readlane( (int)mine, (int)seq );
    } else {
      length = min( a.lengths[seq], a.max_keys );
    }
    b->seq = __builtin_amdgcn_readfirstlane( seq );
    if ( length == 0 ) {
      return false;
    }
    b->row0 = b->seq;
    b->tokens = 1;
    b->start = length - 1;
    return true;
  } else {
    PackedBlock f;
    if ( !packed_block( a.seqs, a.gqa, COLS, number, &f ) ) {
      return false;
    }
    // (said to be the same in every lane: what descriptors and branches are made of stays in scalar registers)
    b->seq = __builtin_amdgcn_readfirstlane( f.seq );
    b->col0 = __builtin_amdgcn_readfirstlane( f.block ) * COLS;
    b->row0 = __builtin_amdgcn_readfirstlane( f.row0 );
    b->tokens = __builtin_amdgcn_readfirstlane( f.tokens );
    b->start = __builtin_amdgcn_readfirstlane( f.start );
    return true;
  }
}

// Block number and kv head of a work-group of packed prompts.  Work-groups go to the 8 XCDs in turn and each has an L2 of its own: where the heads are a multiple
// of 8 a head's blocks go to one of them, which then fetches its rows once.
__device__ __forceinline__ void number_and_head( const Call& a, uint32_t* number, uint32_t* h )
{
  if ( a.n_kv_heads % 8 == 0 ) {
    const uint32_t slot = blockIdx.x >> 3, groups = a.n_kv_heads / 8;
    *number = slot / groups;
    *h = slot % groups * 8 + ( blockIdx.x & 7 );
  } else {
    *number = blockIdx.x / a.n_kv_heads;
    *h = blockIdx.x % a.n_kv_heads;
  }
}

// keys that token t of a block's sequence attends
__device__ __forceinline__ uint32_t visible( const Call& a, const Block& b, uint32_t t ) { return min( b.start + t + 1, a.max_keys ); }

// sum over the lanes that share a column, 16 lanes apart
__device__ __forceinline__ float column_sum( float v ) { return sum_rows( sum_halves( v, v ), sum_halves( v, v ) ); }

// ---- what a masked key's row must not do ---------------------------------------------------------------
// A tile multiplies the values of keys that a column does not attend by a weight of zero, and an infinity or a NaN among them makes a NaN of the sum.  Packed prompts'
// kernels look for columns whose result holds a NaN or an infinity, but not in the sum of the weights (a NaN there is one of an attended key's score, and the whole row is
// NaN).  Where all the values are finite that a column of the wave may have met without attending them, the result is the formula's (an infinite value whose weight is 0
// as the tile has it gives NaN); else those columns are made again here, 16 at a time, by the wave alone and with exact masks.
// 2048 tokens, 8 heads of 128 on one, f16, 53 us a call on its own: with a row of NaN 53 us; with NaN in the values alone of one of the first tokens 57, of one of the last
// (whose wave walks all the keys before it) 580; with infinite values in every row 620.  4096 tokens of 64 heads: 300, 330, 385, 1380 and 3900.

// whether the values of a head are finite in all rows [from, to), by a whole wave
template<typename T>
__device__ __noinline__ bool finite_values( Pages p, uint32_t seq, uint32_t v_off, uint32_t size, uint32_t from, uint32_t to )
{
  const uint32_t lane = threadIdx.x & 63;
  float probe = 0.0f;
  for ( uint32_t key = from; key < to; key++ ) {
    const T* v = reinterpret_cast<const T*>( p.row( seq, key ) ) + v_off;
    for ( uint32_t d = lane; d < size; d += 64 ) {
      probe += 0.0f * to_f32( v[d] );
    }
  }
  return __builtin_amdgcn_ballot_w64( probe != probe ) == 0;
}

// Four neighbouring values of a row of `size`, from d on, 0 behind it, without a branch (a load behind one would be waited for before the next).
// FOURS: the size is a multiple of 4.
template<typename T, bool FOURS>
struct Four
{
  T e[4];
  __device__ __forceinline__ void load( const T* row, uint32_t d, uint32_t size )
  {
    if constexpr ( FOURS ) {
      __builtin_memcpy( e, row + ( d < size ? d : 0 ), sizeof( e ) ); // rows may begin anywhere
    }
#pragma unroll
    for ( uint32_t i = 0; i < 4; i++ ) {
      if constexpr ( !FOURS ) {
        e[i] = row[min( d + i, size - 1 )];
      }
      e[i] = d + i < size ? e[i] : from_f32<T>( 0.0f );
    }
  }
};

// Columns col0 + c of block b, those with bit c of `which` set, over the keys of its split [k_begin, k_most): results put where the tile's are.
// Keys that all of them see in tiles of 16, products in fp32 matrix instructions with operands straight from memory; the others one by one.
template<typename T, int NB, bool FOURS>
__device__ __forceinline__ void columns_again( const T* __restrict__ q, T* __restrict__ out, const Call& a, const Block& b, uint32_t col0, uint32_t which, uint32_t k_begin, uint32_t k_most )
{
  const uint32_t lane = threadIdx.x & 63, c = lane & 15, g4 = lane >> 4, n_heads = a.n_kv_heads * a.gqa;
  const bool ok = which >> c & 1;
  auto end_of = [&]( uint32_t col ) { return min( visible( a, b, col / a.gqa ), k_most ); };
  const uint32_t t_all = end_of( col0 + (uint32_t)__builtin_ctz( which ) ), t_end = end_of( col0 + 31 - (uint32_t)__builtin_clz( which ) );
  const uint32_t col = ok ? col0 + c : col0 + (uint32_t)__builtin_ctz( which ), my_end = end_of( col );
  const uint64_t place = (uint64_t)( b.row0 + col / a.gqa ) * n_heads + b.h * a.gqa + col % a.gqa;
  const uint32_t k_off = b.h * a.size, v_off = ( a.n_kv_heads + b.h ) * a.size;
  auto row = [&]( uint32_t key ) { return reinterpret_cast<const T*>( a.pages.row( b.seq, key ) ); };

  mfma_f32x4 acc[NB]; // element i of acc[n]: dim 16 n + 4 g4 + i of the lane's column
#pragma unroll
  for ( int n = 0; n < NB; n++ ) {
    acc[n] = mfma_f32x4 { 0, 0, 0, 0 };
  }
  float m = -INFINITY, l = 0.0f;
  Four<T, FOURS> x[NB]; // of the query: dims 16 n + 4 g4 ..
#pragma unroll
  for ( int n = 0; n < NB; n++ ) {
    x[n].load( q + place * a.size, 16 * n + 4 * g4, a.size );
  }
  uint32_t t0 = k_begin;
  const T *k_row = row( t0 + min( c, t_end - 1 - t0 ) ), *v_row[4]; // (asked for a tile ahead)
#pragma unroll
  for ( uint32_t i = 0; i < 4; i++ ) {
    v_row[i] = row( t0 + min( 4 * g4 + i, t_end - 1 - t0 ) );
  }
  for ( ; t0 + 16 <= t_all; t0 += 16 ) {
    Four<T, FOURS> k[NB];
    T v[NB][4];
#pragma unroll
    for ( int n = 0; n < NB; n++ ) {
      k[n].load( k_row + k_off, 16 * n + 4 * g4, a.size );
    }
#pragma unroll
    for ( uint32_t n = 0; n < NB; n++ ) {
#pragma unroll
      for ( int i = 0; i < 4; i++ ) {
        v[n][i] = v_row[i][v_off + min( 16 * n + c, a.size - 1 )];
        v[n][i] = 16 * n + c < a.size ? v[n][i] : from_f32<T>( 0.0f );
      }
    }
    const uint32_t ahead = min( t0 + 16, t_end - 1 );
    k_row = row( min( ahead + c, t_end - 1 ) );
#pragma unroll
    for ( uint32_t i = 0; i < 4; i++ ) {
      v_row[i] = row( min( ahead + 4 * g4 + i, t_end - 1 ) );
    }
    mfma_f32x4 st = { 0, 0, 0, 0 };
#pragma unroll
    for ( int n = 0; n < NB; n++ ) {
#pragma unroll
      for ( int e = 0; e < 4; e++ ) {
        st = __builtin_amdgcn_mfma_f32_16x16x4f32( to_f32( k[n].e[e] ), to_f32( x[n].e[e] ), st, 0, 0, 0 );
      }
    }
    float mx = -INFINITY, p[4];
#pragma unroll
    for ( int i = 0; i < 4; i++ ) {
      p[i] = st[i] * a.scale_log2e;
      mx = fmaxf( mx, p[i] );
    }
    mx = fmaxf( mx, __shfl_xor( mx, 16, WAVE ) );
    mx = fmaxf( mx, __shfl_xor( mx, 32, WAVE ) );
    const float m_new = fmaxf( m, mx ), m_safe = m_new == -INFINITY ? 0.0f : m_new, alpha = fast_exp2( m - m_safe );
    m = m_new;
    l *= alpha;
#pragma unroll
    for ( int i = 0; i < 4; i++ ) {
      p[i] = fast_exp2( p[i] - m_safe );
      l += p[i];
    }
#pragma unroll
    for ( int n = 0; n < NB; n++ ) {
      acc[n] *= alpha;
#pragma unroll
      for ( int i = 0; i < 4; i++ ) {
        acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32( to_f32( v[n][i] ), p[i], acc[n], 0, 0, 0 );
      }
    }
  }
  l = column_sum( l );
  for ( ; t0 < t_end; t0++ ) {
    const T* kv = row( t0 );
    Four<T, FOURS> k[NB], v[NB];
    float s = 0.0f;
#pragma unroll
    for ( int n = 0; n < NB; n++ ) {
      k[n].load( kv + k_off, 16 * n + 4 * g4, a.size );
      v[n].load( kv + v_off, 16 * n + 4 * g4, a.size );
    }
#pragma unroll
    for ( int n = 0; n < NB; n++ ) {
#pragma unroll
      for ( int e = 0; e < 4; e++ ) {
        s = __builtin_fmaf( to_f32( x[n].e[e] ), to_f32( k[n].e[e] ), s );
      }
    }
    s = column_sum( s ) * a.scale_log2e;
    if ( t0 < my_end ) {
      const float m_new = fmaxf( m, s ), m_safe = m_new == -INFINITY ? 0.0f : m_new, alpha = fast_exp2( m - m_safe ), w = fast_exp2( s - m_safe );
      m = m_new;
      l = __builtin_fmaf( l, alpha, w );
#pragma unroll
      for ( int n = 0; n < NB; n++ ) {
#pragma unroll
        for ( int i = 0; i < 4; i++ ) {
          acc[n][i] = __builtin_fmaf( w, to_f32( v[n].e[i] ), acc[n][i] * alpha );
        }
      }
    }
  }
  if ( !ok ) {
    return;
  }
  const uint64_t slot = place * a.splits + b.split;
#pragma unroll
  for ( int n = 0; n < NB; n++ ) {
#pragma unroll
    for ( int i = 0; i < 4; i++ ) {
      const uint32_t d = 16 * n + 4 * g4 + i;
      if ( d < a.size ) {
        if ( a.splits == 1 ) {
          out[place * a.size + d] = from_f32<T>( acc[n][i] / l );
        } else {
          a.part_out[slot * a.size + d] = acc[n][i];
        }
      }
    }
  }
  if ( a.splits > 1 && g4 == 0 ) {
    a.part_ml[slot * 2] = m;
    a.part_ml[slot * 2 + 1] = l;
  }
}

// `which`: columns of a wave, which is through with storing results; masked: the first key that some column of the wave does not see, end: behind those of the work-group.
// A function of its own so that the kernels' registers are not divided otherwise for it (inline it cost 3 to 25 %), and one for each kernel, since a function is
// given the fewest registers of its callers': KERNEL tells them apart.
template<typename T, int NB, bool FOURS, int KERNEL>
__device__ __noinline__ void masked_again( const T* q, T* out, Call a, Block b, uint32_t col0, uint32_t which, uint32_t k_begin, uint32_t k_most, uint32_t masked, uint32_t end )
{
  if ( finite_values<T>( a.pages, b.seq, ( a.n_kv_heads + b.h ) * a.size, a.size, max( k_begin, masked ), end ) ) {
    return;
  }
  __builtin_amdgcn_s_waitcnt( 0x0F70 ); // vmcnt(0): the results that are written again have been written
  for ( ; which != 0; col0 += 16, which >>= 16 ) {
    if ( ( which & 0xffff ) != 0 ) {
      columns_again<T, NB, FOURS>( q, out, a, b, col0, which & 0xffff, k_begin, k_most );
    }
  }
}

template<typename T>
struct alignas( 4 * sizeof( T ) ) Piece
{
  T e[4];
};

// =================================================================================================
// tile kernel in fp32: any storage type, head size up to 16 NB, page size, alignment
//
// Keys and values of a stage go to LDS as fp32 (zeros behind the head and behind the keys), scores and sums are products of the fp32 matrix instruction
// (16 x 16, 4 deep, 256 operations a cycle and CU): S^T = K Q^T with a lane's queries in registers, then O^T += V^T P^T, whose second operand is the
// scores' result as it lies (lane (g, c): keys 4 g + i of column c); a column's maximum and sum stay in the lanes of its c.
//   packed: 64 columns a work-group, 16 a wave, stages of 32 keys that all four waves go through
//   decode: 16 columns, stages of 64 keys, 16 a wave, the four joined through LDS at the end
// The next stage's rows are asked for before a stage is computed.
// Taken where rows cannot go straight to LDS in pieces of 16 bytes: head sizes that are no multiple of them, pages below 16 tokens, pool or rows that are not aligned.
// Bound by its own conversions and LDS traffic.  f16, 8 heads on 4 kv heads of 36: decode of 64 contexts of 100 to 4000 keys 94 us (0.8 TB/s; heads of 40 in the streaming
// kernel 45), a prompt of 4000 tokens 376 us (53).
// =================================================================================================
template<typename T, int NB, bool DECODE>
__global__ __launch_bounds__( 256, DECODE || NB == 16 ? 1 : NB == 8 ? 2 : 3 ) void attn_pages_f32_kernel( const T* __restrict__ q, T* __restrict__ out, Call a )
{
  constexpr uint32_t HSP = 16 * NB, LD = HSP + 4, KEYS = DECODE ? 64 : 32, COLS = DECODE ? 16 : 64;
  constexpr uint32_t VR = HSP / 4;                     // pieces of a padded head
  constexpr uint32_t ROWS = 256 / VR;                  // keys that the work-group takes at once
  constexpr uint32_t U = KEYS / ROWS;                  // pieces a thread takes of K, and of V
  __shared__ float s_k[KEYS * LD], s_v[KEYS * LD];

  const uint32_t wave = __builtin_amdgcn_readfirstlane( threadIdx.x >> 6 ), lane = threadIdx.x & 63, c = lane & 15, g4 = lane >> 4;
  Block b;
  if ( !block_of<DECODE, COLS>( a, blockIdx.x, blockIdx.y, blockIdx.z, &b ) ) {
    return;
  }
  const uint32_t n_heads = a.n_kv_heads * a.gqa, n_cols = b.tokens * a.gqa;
  const uint32_t last_col = min( n_cols, b.col0 + COLS ) - 1;
  const uint32_t k_begin = b.split * a.chunk, k_end = min( visible( a, b, last_col / a.gqa ), k_begin + a.chunk );
  if ( k_begin >= k_end ) {
    return;
  }
  const uint32_t col = b.col0 + ( DECODE ? 0 : 16 * wave ) + c;
  const bool ok = col < n_cols;
  const uint32_t token = ok ? col / a.gqa : 0, head = b.h * a.gqa + ( ok ? col % a.gqa : 0 );
  const uint64_t qrow = ( (uint64_t)( b.row0 + token ) * n_heads + head ) * a.size;
  const uint32_t my_end = ok ? min( visible( a, b, token ), k_end ) : 0; // keys this column attends here: [k_begin, my_end)
  const uint32_t kv_off = b.h * a.size, v_off = ( a.n_kv_heads + b.h ) * a.size;
  const bool whole = a.size % 4 == 0
                     && ( ( reinterpret_cast<uintptr_t>( a.pages.pool ) | a.pages.stride | reinterpret_cast<uintptr_t>( q ) | reinterpret_cast<uintptr_t>( out ) ) & ( 4 * sizeof( T ) - 1 ) ) == 0;

  // queries: dims 16 s + 4 g4 + e of the lane's column
  float qd[NB][4];
#pragma unroll
  for ( int s = 0; s < NB; s++ ) {
#pragma unroll
    for ( int e = 0; e < 4; e++ ) {
      const uint32_t d = 16 * s + 4 * g4 + e;
      qd[s][e] = ok && d < a.size ? to_f32( q[qrow + d] ) : 0.0f;
    }
  }

  mfma_f32x4 acc[NB]; // element i of acc[n]: dim 16 n + 4 g4 + i of the lane's column
#pragma unroll
  for ( int n = 0; n < NB; n++ ) {
    acc[n] = mfma_f32x4 { 0, 0, 0, 0 };
  }
  float m = -INFINITY, l = 0.0f; // l: of this lane's keys

  const uint32_t my_piece = threadIdx.x % VR, my_row = threadIdx.x / VR;
  Piece<T> kn[U], vn[U];
  auto fetch = [&]( uint32_t t0 ) __attribute__( ( always_inline ) ) {
#pragma unroll
    for ( uint32_t u = 0; u < U; u++ ) {
      const uint32_t key = t0 + u * ROWS + my_row;
#pragma unroll
      for ( int e = 0; e < 4; e++ ) {
        kn[u].e[e] = vn[u].e[e] = from_f32<T>( 0.0f );
      }
      if ( key < k_end && 4 * my_piece < a.size ) {
        const T* row = reinterpret_cast<const T*>( a.pages.row( b.seq, key ) ) + 4 * my_piece;
        if ( whole ) {
          kn[u] = *reinterpret_cast<const Piece<T>*>( row + kv_off );
          vn[u] = *reinterpret_cast<const Piece<T>*>( row + v_off );
        } else {
#pragma unroll
          for ( int e = 0; e < 4; e++ ) {
            if ( 4 * my_piece + e < a.size ) {
              kn[u].e[e] = row[kv_off + e];
              vn[u].e[e] = row[v_off + e];
            }
          }
        }
      }
    }
  };
  fetch( k_begin );
  for ( uint32_t t0 = k_begin; t0 < k_end; t0 += KEYS ) {
    __syncthreads(); // every wave is done with the stage before
#pragma unroll
    for ( uint32_t u = 0; u < U; u++ ) {
      float* k = s_k + ( u * ROWS + my_row ) * LD + 4 * my_piece;
      float* v = s_v + ( u * ROWS + my_row ) * LD + 4 * my_piece;
#pragma unroll
      for ( int e = 0; e < 4; e++ ) {
        k[e] = to_f32( kn[u].e[e] );
        v[e] = to_f32( vn[u].e[e] );
      }
    }
    __syncthreads();
    if ( t0 + KEYS < k_end ) {
      fetch( t0 + KEYS );
    }
    constexpr int TILES = DECODE ? 1 : KEYS / 16;
#pragma unroll
    for ( int tile = 0; tile < TILES; tile++ ) {
      const uint32_t r0 = DECODE ? 16 * wave : 16 * tile; // first key of the tile within the stage
      mfma_f32x4 st = { 0, 0, 0, 0 };
#pragma unroll
      for ( int s = 0; s < NB; s++ ) {
        const float4 k = *reinterpret_cast<const float4*>( s_k + ( r0 + c ) * LD + 16 * s + 4 * g4 );
        st = __builtin_amdgcn_mfma_f32_16x16x4f32( k.x, qd[s][0], st, 0, 0, 0 );
        st = __builtin_amdgcn_mfma_f32_16x16x4f32( k.y, qd[s][1], st, 0, 0, 0 );
        st = __builtin_amdgcn_mfma_f32_16x16x4f32( k.z, qd[s][2], st, 0, 0, 0 );
        st = __builtin_amdgcn_mfma_f32_16x16x4f32( k.w, qd[s][3], st, 0, 0, 0 );
      }
      float p[4], mx = -INFINITY;
#pragma unroll
      for ( int i = 0; i < 4; i++ ) {
        p[i] = t0 + r0 + 4 * g4 + i < my_end ? st[i] * a.scale_log2e : -INFINITY;
        mx = fmaxf( mx, p[i] );
      }
      mx = fmaxf( mx, __shfl_xor( mx, 16, WAVE ) );
      mx = fmaxf( mx, __shfl_xor( mx, 32, WAVE ) );
      const float m_new = fmaxf( m, mx ), m_safe = m_new == -INFINITY ? 0.0f : m_new;
      const float alpha = fast_exp2( m - m_safe );
      m = m_new;
#pragma unroll
      for ( int i = 0; i < 4; i++ ) {
        p[i] = fast_exp2( p[i] - m_safe );
      }
      l = l * alpha + ( ( p[0] + p[1] ) + ( p[2] + p[3] ) );
      if ( __builtin_amdgcn_ballot_w64( alpha != 1.0f ) != 0 ) {
#pragma unroll
        for ( int n = 0; n < NB; n++ ) {
          acc[n] *= alpha;
        }
      }
#pragma unroll
      for ( int n = 0; n < NB; n++ ) {
#pragma unroll
        for ( int i = 0; i < 4; i++ ) {
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32( s_v[( r0 + 4 * g4 + i ) * LD + 16 * n + c], p[i], acc[n], 0, 0, 0 );
        }
      }
    }
  }
  l += __shfl_xor( l, 16, WAVE );
  l += __shfl_xor( l, 32, WAVE );

  if constexpr ( DECODE ) {
    // the four waves' parts added up by wave 0, lane for lane as they lie in the registers; s_v holds them
    static_assert( 3 * 64 * ( 4 * NB + 2 ) <= KEYS * LD, "the parts fit" );
    __syncthreads();
    if ( wave != 0 ) {
      float* part = s_v + ( wave - 1 ) * 64 * ( 4 * NB + 2 );
      part[lane] = m;
      part[64 + lane] = l;
#pragma unroll
      for ( int n = 0; n < NB; n++ ) {
#pragma unroll
        for ( int i = 0; i < 4; i++ ) {
          part[( 2 + 4 * n + i ) * 64 + lane] = acc[n][i];
        }
      }
    }
    __syncthreads();
    if ( wave != 0 ) {
      return;
    }
    float mm = m;
    for ( int w = 0; w < 3; w++ ) {
      mm = fmaxf( mm, s_v[w * 64 * ( 4 * NB + 2 ) + lane] );
    }
    const float mm_safe = mm == -INFINITY ? 0.0f : mm, w0 = fast_exp2( m - mm_safe );
    m = mm;
    l *= w0;
#pragma unroll
    for ( int n = 0; n < NB; n++ ) {
      acc[n] *= w0;
    }
    for ( int w = 0; w < 3; w++ ) {
      const float* part = s_v + w * 64 * ( 4 * NB + 2 );
      const float ww = fast_exp2( part[lane] - mm_safe );
      l = __builtin_fmaf( part[64 + lane], ww, l );
#pragma unroll
      for ( int n = 0; n < NB; n++ ) {
#pragma unroll
        for ( int i = 0; i < 4; i++ ) {
          acc[n][i] = __builtin_fmaf( part[( 2 + 4 * n + i ) * 64 + lane], ww, acc[n][i] );
        }
      }
    }
  }

  const uint64_t place = (uint64_t)( b.row0 + token ) * n_heads + head; // of the (row, head) among the outputs
  const uint64_t slot = place * a.splits + b.split;
  const bool mine = ok && k_begin < my_end;
  if ( mine && a.splits > 1 ) {
#pragma unroll
    for ( int n = 0; n < NB; n++ ) {
#pragma unroll
      for ( int i = 0; i < 4; i++ ) {
        const uint32_t d = 16 * n + 4 * g4 + i;
        if ( d < a.size ) {
          a.part_out[slot * a.size + d] = acc[n][i];
        }
      }
    }
    if ( g4 == 0 ) {
      a.part_ml[slot * 2] = m;
      a.part_ml[slot * 2 + 1] = l;
    }
  } else if ( mine ) {
    const float inv = 1.0f / l;
#pragma unroll
    for ( int n = 0; n < NB; n++ ) {
      const uint32_t d = 16 * n + 4 * g4;
      if ( whole ) {
        if ( d < a.size ) {
          Piece<T> o;
#pragma unroll
          for ( int i = 0; i < 4; i++ ) {
            o.e[i] = from_f32<T>( acc[n][i] * inv );
          }
          *reinterpret_cast<Piece<T>*>( out + place * a.size + d ) = o;
        }
      } else {
#pragma unroll
        for ( int i = 0; i < 4; i++ ) {
          if ( d + i < a.size ) {
            out[place * a.size + d + i] = from_f32<T>( acc[n][i] * inv );
          }
        }
      }
    }
  }
  if constexpr ( !DECODE ) {
    float probe = 0.0f;
#pragma unroll
    for ( int n = 0; n < NB; n++ ) {
      probe += 0.0f * ( ( acc[n][0] + acc[n][1] ) + ( acc[n][2] + acc[n][3] ) );
    }
    const uint64_t lanes = __builtin_amdgcn_ballot_w64( mine && probe != probe && l == l );
    const uint32_t bad = (uint32_t)( lanes | lanes >> 16 | lanes >> 32 | lanes >> 48 ) & 0xffff; // columns
    if ( bad != 0 ) {
      const uint32_t first_col = b.col0 + 16 * wave;
      masked_again<T, NB, false, 0>( q, out, a, b, first_col, bad, k_begin, k_begin + a.chunk, min( visible( a, b, first_col / a.gqa ), k_end ), k_end );
    }
  }
}

// =================================================================================================
// decode, heads of up to CH chunks of 16 bytes: wave <-> (context, kv head, 16 columns, run of keys)
//
// Bound by the bytes of the cache.  A wave goes through stages of 32 keys on its own: their K and V rows go from memory straight to its part of LDS, two stages deep,
// so that a stage (16 KB at 128 16-bit elements) is always on its way while one is computed.  Rows behind the keys, and chunks behind a smaller head, lie outside the
// descriptor of their 16 rows (which lie in one page) and arrive as zeros, whatever memory holds there.
//   S^T = K Q^T     16 x 16 x 32: a lane gets keys 4 g + i (and 16 + 4 g + i) of column c
//   O^T += V^T P^T  16 x 16 x 32: the weights are the second operand as they lie, if slot 8 g + e is key 4 g + e (e < 4) and 16 + 4 g + e - 4; the first operand's
//                   lanes take those keys of one dim with transposing LDS reads
// 16-byte chunks of a row are swizzled by the row (in the address a lane fetches) so that both reads touch every bank once.
// The weights are rounded to the storage type for the second product, as the matrix units take them; the sum takes them rounded too.  (In two parts, a second product or
// the columns that up to 8 queries leave free, the error against 64 bits is the plain form's, 2.1e-4 for 2.7e-4 in f16, and 1.7e-3 for 2.4e-3 in bf16; 1 context of 301 keys
// takes 7.2 us for 7.0, 16 of 500 9.7 for 9.4.)  An infinite value whose weight rounds to 0 makes NaN.
// fp32: both products 16 x 16 x 4, a chunk of K being four of its steps, weights as they are, and V read value by value; 16 keys a stage above 64 elements.
// (64 contexts of 100 to 4000 keys, 8 heads of 256 in fp32: 357 us, 6.0 TB/s; in the tile kernel above 1530.)
// W waves of a work-group take the stages of one run in turns and are joined through LDS.
// f16, 8 kv heads of 128 with 8 queries each: 64 contexts of 57 to 4096 keys 90 us (6.0 TB/s), 1 of 301 keys 7.0 us, of which a launch that only stores takes 3;
// bf16, 32 heads, 3 contexts of 20011 to 32768 keys: 226 us (5.7 TB/s), the launch that joins the splits (4.8) among them.
// =================================================================================================
typedef __attribute__( ( address_space( 3 ) ) ) void* lds_ptr;
typedef __attribute__( ( address_space( 3 ) ) ) char lds_char;
typedef short v4s __attribute__( ( ext_vector_type( 4 ) ) );
typedef short v8s __attribute__( ( ext_vector_type( 8 ) ) );
typedef __attribute__( ( address_space( 3 ) ) ) v4s* lds_v4s;

constexpr float LAZY = 8.0f; // the reference point of the exponentials stays until a maximum is 2^LAZY above it: fewer rescalings
// The reference point lies so many powers of two below the maximum it was taken from.  f16 weights then go up to 2^15, and what rounds to 0 is below 2^-32 of the largest
// (at 0 it would be 2^-25, and the weights of a long context next to one key far above it would be lost).
template<typename E>
constexpr float LIFT = std::is_same_v<E, __half> ? 7.0f : 0.0f;

// maximum over the lanes that share a column, 16 lanes apart, without a trip through LDS
[[maybe_unused]] __device__ __forceinline__ float column_max( float v )
{
  v = half_wave_max( v );
  const unsigned bits = __builtin_bit_cast( unsigned, v );
  const auto r = __builtin_amdgcn_permlane16_swap( bits, bits, false, false );
  const unsigned r0 = r[0], r1 = r[1];
  return fmaxf( __builtin_bit_cast( float, r0 ), __builtin_bit_cast( float, r1 ) );
}

// a weight as the storage type holds it
template<typename E>
__device__ __forceinline__ float rounded( float v )
{
  return to_f32( from_f32<E>( v ) );
}

template<typename E>
struct ChunkOf // 16 bytes as the matrix instructions take them
{
  using type = typename Mfma<E>::x8;
};
template<>
struct ChunkOf<float>
{
  using type = mfma_f32x4;
};

// four neighbouring values of a row, aligned to them
template<typename E>
__device__ __forceinline__ void store4( E* to, float a, float b, float c, float d )
{
  if constexpr ( sizeof( E ) == 4 ) {
    *reinterpret_cast<float4*>( to ) = make_float4( a, b, c, d );
  } else {
    *reinterpret_cast<uint2*>( to ) = make_uint2( rounded_pair<E>( a, b ), rounded_pair<E>( c, d ) );
  }
}

template<uint32_t FIRST, typename Chunk>
__device__ __forceinline__ void read_chunks( const uint32_t* at, Chunk* k )
{
  asm volatile( "ds_read_b128 %0, %8 offset:%16\n\t"
                "ds_read_b128 %1, %9 offset:%16\n\t"
                "ds_read_b128 %2, %10 offset:%16\n\t"
                "ds_read_b128 %3, %11 offset:%16\n\t"
                "ds_read_b128 %4, %12 offset:%16\n\t"
                "ds_read_b128 %5, %13 offset:%16\n\t"
                "ds_read_b128 %6, %14 offset:%16\n\t"
                "ds_read_b128 %7, %15 offset:%16\n\t"
                "s_waitcnt lgkmcnt(0)"
                : "=&v"( k[0] ), "=&v"( k[1] ), "=&v"( k[2] ), "=&v"( k[3] ), "=&v"( k[4] ), "=&v"( k[5] ), "=&v"( k[6] ), "=&v"( k[7] )
                : "v"( at[0] ), "v"( at[1] ), "v"( at[2] ), "v"( at[3] ), "v"( at[4] ), "v"( at[5] ), "v"( at[6] ), "v"( at[7] ), "n"( FIRST )
                : "memory" );
}

// LDS reads of a stage, written out, each block with its waits: the compiler cannot tell the tiles that a read may take from the ones on their way, and would wait
// for all of them.
template<int CH, uint32_t FIRST, uint32_t SECOND, typename Chunk, uint32_t NU>
__device__ __forceinline__ void read_keys( const uint32_t* at, Chunk ( &k )[NU][CH / 4] )
{
  if constexpr ( CH == 64 ) {
    static_assert( NU == 1, "" );
    asm volatile( "s_waitcnt vmcnt(32)" ::: "memory" );
    read_chunks<FIRST>( at, k[0] );
    read_chunks<FIRST>( at + 8, k[0] + 8 );
  } else if constexpr ( CH == 32 ) {
    if constexpr ( NU == 1 ) {
      asm volatile( "s_waitcnt vmcnt(16)" ::: "memory" );
    } else {
      asm volatile( "s_waitcnt vmcnt(32)" ::: "memory" );
    }
    read_chunks<FIRST>( at, k[0] );
    if constexpr ( NU == 2 ) {
      read_chunks<SECOND>( at, k[1] );
    }
  } else if constexpr ( CH == 16 ) {
    asm volatile( "s_waitcnt vmcnt(16)\n\t"
                  "ds_read_b128 %0, %8 offset:%12\n\t"
                  "ds_read_b128 %1, %9 offset:%12\n\t"
                  "ds_read_b128 %2, %10 offset:%12\n\t"
                  "ds_read_b128 %3, %11 offset:%12\n\t"
                  "ds_read_b128 %4, %8 offset:%13\n\t"
                  "ds_read_b128 %5, %9 offset:%13\n\t"
                  "ds_read_b128 %6, %10 offset:%13\n\t"
                  "ds_read_b128 %7, %11 offset:%13\n\t"
                  "s_waitcnt lgkmcnt(0)"
                  : "=&v"( k[0][0] ), "=&v"( k[0][1] ), "=&v"( k[0][2] ), "=&v"( k[0][3] ), "=&v"( k[1][0] ), "=&v"( k[1][1] ), "=&v"( k[1][2] ), "=&v"( k[1][3] )
                  : "v"( at[0] ), "v"( at[1] ), "v"( at[2] ), "v"( at[3] ), "n"( FIRST ), "n"( SECOND )
                  : "memory" );
  } else {
    asm volatile( "s_waitcnt vmcnt(8)\n\t"
                  "ds_read_b128 %0, %4 offset:%6\n\t"
                  "ds_read_b128 %1, %5 offset:%6\n\t"
                  "ds_read_b128 %2, %4 offset:%7\n\t"
                  "ds_read_b128 %3, %5 offset:%7\n\t"
                  "s_waitcnt lgkmcnt(0)"
                  : "=&v"( k[0][0] ), "=&v"( k[0][1] ), "=&v"( k[1][0] ), "=&v"( k[1][1] )
                  : "v"( at[0] ), "v"( at[1] ), "n"( FIRST ), "n"( SECOND )
                  : "memory" );
  }
}
// four blocks of 16 dims
template<uint32_t FIRST, uint32_t SECOND>
__device__ __forceinline__ void read_values( const uint32_t* at, v4s ( *v )[2] )
{
  asm volatile( "ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
                "ds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                "ds_read_b64_tr_b16 %2, %9 offset:%12\n\t"
                "ds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                "ds_read_b64_tr_b16 %4, %10 offset:%12\n\t"
                "ds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                "ds_read_b64_tr_b16 %6, %11 offset:%12\n\t"
                "ds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                "s_waitcnt lgkmcnt(0)"
                : "=&v"( v[0][0] ), "=&v"( v[0][1] ), "=&v"( v[1][0] ), "=&v"( v[1][1] ), "=&v"( v[2][0] ), "=&v"( v[2][1] ), "=&v"( v[3][0] ), "=&v"( v[3][1] )
                : "v"( at[0] ), "v"( at[1] ), "v"( at[2] ), "v"( at[3] ), "n"( FIRST ), "n"( SECOND )
                : "memory" );
}

// a lane's chunk of eight groups of rows, 1 KB apart
template<uint32_t FIRST, bool WAIT>
__device__ __forceinline__ void read_rows( uint32_t at, mfma_f32x4 ( &v )[8] )
{
  if constexpr ( WAIT ) {
    asm volatile( "s_waitcnt vmcnt(16)" ::: "memory" );
  }
  asm volatile( "ds_read_b128 %0, %8 offset:%9\n\t"
                "ds_read_b128 %1, %8 offset:%10\n\t"
                "ds_read_b128 %2, %8 offset:%11\n\t"
                "ds_read_b128 %3, %8 offset:%12\n\t"
                "ds_read_b128 %4, %8 offset:%13\n\t"
                "ds_read_b128 %5, %8 offset:%14\n\t"
                "ds_read_b128 %6, %8 offset:%15\n\t"
                "ds_read_b128 %7, %8 offset:%16\n\t"
                "s_waitcnt lgkmcnt(0)"
                : "=&v"( v[0] ), "=&v"( v[1] ), "=&v"( v[2] ), "=&v"( v[3] ), "=&v"( v[4] ), "=&v"( v[5] ), "=&v"( v[6] ), "=&v"( v[7] )
                : "v"( at ), "n"( FIRST ), "n"( FIRST + 1 * 1024 ), "n"( FIRST + 2 * 1024 ), "n"( FIRST + 3 * 1024 ), "n"( FIRST + 4 * 1024 ), "n"( FIRST + 5 * 1024 ), "n"( FIRST + 6 * 1024 ),
                  "n"( FIRST + 7 * 1024 )
                : "memory" );
}

// A stage's values as the first operand of O^T += V^T P^T
template<typename E, uint32_t NB, uint32_t NU>
struct Values
{
  v4s half[NB][2];
  template<int CH, uint32_t FIRST, uint32_t SECOND>
  __device__ __forceinline__ void read( const uint32_t* at )
  {
#pragma unroll
    for ( uint32_t n = 0; n < NB; n += 4 ) {
      read_values<FIRST, SECOND>( at + n, half + n );
    }
  }
  __device__ __forceinline__ void add( const float* p, mfma_f32x4 ( &acc )[NB] ) const
  {
    typedef uint32_t u32x4 __attribute__( ( ext_vector_type( 4 ) ) );
    using X8 = typename Mfma<E>::x8;
    const X8 pk = __builtin_bit_cast( X8, ( u32x4 { rounded_pair<E>( p[0], p[1] ), rounded_pair<E>( p[2], p[3] ), rounded_pair<E>( p[4], p[5] ), rounded_pair<E>( p[6], p[7] ) } ) );
#pragma unroll
    for ( uint32_t n = 0; n < NB; n++ ) {
      const v8s v = v8s { half[n][0][0], half[n][0][1], half[n][0][2], half[n][0][3], half[n][1][0], half[n][1][1], half[n][1][2], half[n][1][3] };
      acc[n] = Mfma<E>::k32( __builtin_bit_cast( X8, v ), pk, acc[n] );
    }
  }
};
// eight values of fp32 rows 16 CH bytes apart: of four rows and the four 16 rows on, or of four rows at two addresses
template<int CH, uint32_t FIRST, bool TWO>
__device__ __forceinline__ void read_values_f32( const uint32_t* at, float* v )
{
  constexpr uint32_t ROW = CH * 16, NEXT = TWO ? FIRST : FIRST + 16 * ROW;
  asm volatile( "ds_read_b32 %0, %8 offset:%10\n\t"
                "ds_read_b32 %1, %8 offset:%11\n\t"
                "ds_read_b32 %2, %8 offset:%12\n\t"
                "ds_read_b32 %3, %8 offset:%13\n\t"
                "ds_read_b32 %4, %9 offset:%14\n\t"
                "ds_read_b32 %5, %9 offset:%15\n\t"
                "ds_read_b32 %6, %9 offset:%16\n\t"
                "ds_read_b32 %7, %9 offset:%17\n\t"
                "s_waitcnt lgkmcnt(0)"
                : "=&v"( v[0] ), "=&v"( v[1] ), "=&v"( v[2] ), "=&v"( v[3] ), "=&v"( v[4] ), "=&v"( v[5] ), "=&v"( v[6] ), "=&v"( v[7] )
                : "v"( at[0] ), "v"( at[TWO ? 1 : 0] ), "n"( FIRST ), "n"( FIRST + ROW ), "n"( FIRST + 2 * ROW ), "n"( FIRST + 3 * ROW ), "n"( NEXT ), "n"( NEXT + ROW ),
                  "n"( NEXT + 2 * ROW ), "n"( NEXT + 3 * ROW )
                : "memory" );
}
template<uint32_t NB, uint32_t NU>
struct Values<float, NB, NU>
{
  float v[NB][NU][4];
  template<int CH, uint32_t FIRST, uint32_t SECOND>
  __device__ __forceinline__ void read( const uint32_t* at )
  {
#pragma unroll
    for ( uint32_t n = 0; n < NB; n += 3 - NU ) {
      read_values_f32<CH, FIRST, NU == 1>( at + n, &v[n][0][0] );
    }
  }
  __device__ __forceinline__ void add( const float* p, mfma_f32x4 ( &acc )[NB] ) const
  {
#pragma unroll
    for ( uint32_t u = 0; u < NU; u++ ) {
#pragma unroll
      for ( uint32_t i = 0; i < 4; i++ ) {
#pragma unroll
        for ( uint32_t n = 0; n < NB; n++ ) {
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32( v[n][u][i], p[4 * u + i], acc[n], 0, 0, 0 );
        }
      }
    }
  }
};

template<typename E, int CH, int W, int HW>
__device__ __forceinline__ void decode_run( const E* __restrict__ q, E* __restrict__ out, const Call& a )
{
  constexpr bool F32 = sizeof( E ) == 4;
  constexpr uint32_t PER = 16 / sizeof( E );                    // elements of a chunk
  constexpr uint32_t KEYS = F32 && CH >= 32 ? 16 : 32;          // of a stage
  constexpr uint32_t KK = CH / 4, NB = CH * PER / 16;           // chunks of a key that a lane reads, blocks of 16 dims
  constexpr uint32_t NU = KEYS / 16;
  constexpr uint32_t RPI = 64 / CH;            // rows that a load of the wave fetches
  constexpr uint32_t IPG = 16 / RPI;           // loads for 16 rows of K, or of V
  using Chunk = typename ChunkOf<E>::type;
  constexpr uint32_t TILE = KEYS * CH * 16;    // bytes
  static_assert( W == 1 || HW == 1, "" );
  __shared__ uint4 s_tiles[W * HW][4][KEYS * CH]; // of every wave: K of even and of odd stages, V of even and of odd stages

  const uint32_t wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane( threadIdx.x >> 6 ), lane = threadIdx.x & 63, c = lane & 15, g4 = lane >> 4;
  Block b;
  const uint32_t pairs = a.n_kv_heads / HW, hw = HW == 1 ? 0 : __builtin_amdgcn_readfirstlane( threadIdx.x >> 6 );
  if ( !block_of<true, 16>( a, blockIdx.x / pairs, blockIdx.x % pairs * HW + hw, blockIdx.y, &b ) ) {
    return;
  }
  const uint32_t length = b.start + 1, k_begin = b.split * a.chunk, k_end = min( length, k_begin + a.chunk );
  if ( k_begin >= k_end ) {
    return;
  }
  const uint32_t col = b.col0 + c;
  const bool ok = col < a.gqa;
  const uint64_t place = (uint64_t)b.row0 * a.n_kv_heads * a.gqa + (uint64_t)b.h * a.gqa + ( ok ? col : 0 );

  uint4( *const tiles )[KEYS * CH] = s_tiles[wave + hw];
  Chunk qb[KK];
#pragma unroll
  for ( uint32_t kk = 0; kk < KK; kk++ ) {
    const uint32_t d = PER * ( 4 * kk + g4 );
    qb[kk] = ok && d < a.size ? *reinterpret_cast<const Chunk*>( q + place * a.size + d ) : Chunk {};
  }

  // a lane's place in the rows of a load: row lane / CH, slot lane % CH, which keeps chunk slot ^ (swizzle of the row)
  const uint32_t ld_row = lane / CH, ld_slot = lane % CH, chunks = a.size / PER;
  const uint32_t k_off = b.h * a.size * sizeof( E ), v_off = ( a.n_kv_heads + b.h ) * a.size * sizeof( E );
  auto k_swizzle = []( uint32_t row ) { return CH >= 16 ? row & 15 : ( row >> 1 ) & 7; };
  auto v_swizzle = []( uint32_t row ) { return F32 ? row & 12 : CH >= 16 ? 2 * ( row & 7 ) : 2 * ( ( row >> 1 ) & 3 ); };
  uint32_t k_at[IPG], v_at[IPG];
#pragma unroll
  for ( uint32_t t = 0; t < IPG; t++ ) {
    const uint32_t row = RPI * t + ld_row, kc = ld_slot ^ k_swizzle( row ), vc = ld_slot ^ v_swizzle( row );
    k_at[t] = kc < chunks ? row * a.pages.row_bytes + k_off + 16 * kc : 0x80000000u; // far outside every descriptor
    v_at[t] = vc < chunks ? row * a.pages.row_bytes + v_off + 16 * vc : 0x80000000u;
  }

  const uint32_t n_stages = ( k_end - k_begin + KEYS - 1 ) / KEYS, n_mine = n_stages > wave ? ( n_stages - wave + W - 1 ) / W : 0;
  // Page numbers are read by scalar loads one stage before they are needed: vector loads would be counted with the loads to LDS, and waiting for one would be
  // waiting for those.
  typedef const uint32_t __attribute__( ( address_space( 4 ) ) ) * scalar_ptr;
  const scalar_ptr table = (scalar_ptr)( reinterpret_cast<uintptr_t>( a.pages.table + (uint64_t)b.seq * a.pages.table_stride ) );
  uint32_t id[NU];
  auto look_up = [&]( uint32_t stage ) __attribute__( ( always_inline ) ) {
#pragma unroll
    for ( uint32_t u = 0; u < NU; u++ ) {
      id[u] = table[min( k_begin + KEYS * ( stage * W + wave ) + 16 * u, k_end - 1 ) >> a.pages.shift];
    }
  };
  __amdgpu_buffer_rsrc_t rsrc[NU];
  auto describe = [&]( uint32_t stage ) __attribute__( ( always_inline ) ) {
#pragma unroll
    for ( uint32_t u = 0; u < NU; u++ ) {
      const uint32_t key = k_begin + KEYS * ( stage * W + wave ) + 16 * u;
      const char* base = a.pages.pool + min( id[u], a.pages.last ) * a.pages.stride + (uint64_t)( key & ( ( 1u << a.pages.shift ) - 1 ) ) * a.pages.row_bytes;
      const uint32_t rows = key < k_end ? min( k_end - key, 16u ) : 0u;
      rsrc[u] = __builtin_amdgcn_make_buffer_rsrc( const_cast<char*>( base ), 0, (int)( rows * a.pages.row_bytes ), 0x00020000 );
    }
    look_up( stage + 1 );
  };
  auto fetch = [&]( uint4* tile, const uint32_t( &at )[IPG] ) __attribute__( ( always_inline ) ) {
#pragma unroll
    for ( uint32_t u = 0; u < NU; u++ ) {
#pragma unroll
      for ( uint32_t t = 0; t < IPG; t++ ) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds( rsrc[u], (lds_ptr)( tile + ( 16 * u + RPI * t ) * CH ), 16, at[t], 0, 0, 2 ); // (read once: streaming)
      }
    }
  };

  mfma_f32x4 acc[NB]; // element i of acc[n]: dim 16 n + 4 g4 + i of column c
#pragma unroll
  for ( uint32_t n = 0; n < NB; n++ ) {
    acc[n] = mfma_f32x4 { 0, 0, 0, 0 };
  }
  float m = -INFINITY, l = 0.0f; // l: of this lane's keys

  // K: row c (and row 16 + c), chunk 4 kk + g4.  V in 16 bits, transposing: lane 4 e + p of 16 points at dims 4 p .. 4 p + 3 of key 4 g4 + e and receives
  // one dim of the four keys.  V in fp32: dim c of a block, of keys 4 g4 + i.
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)&tiles[0][0];
  uint32_t k_lds[KK], v_lds[NB];
#pragma unroll
  for ( uint32_t kk = 0; kk < KK; kk++ ) {
    k_lds[kk] = lds0 + c * CH * 16 + ( ( 4 * kk + g4 ) ^ k_swizzle( c ) ) * 16;
  }
  const uint32_t tr_row = 4 * g4 + ( c >> 2 ), tr_at = tr_row * CH * 16 + ( ( ( c & 3 ) >> 1 ) ^ v_swizzle( tr_row ) ) * 16 + ( c & 1 ) * 8;
#pragma unroll
  for ( uint32_t n = 0; n < NB; n++ ) {
    v_lds[n] = lds0 + ( F32 ? 4 * g4 * CH * 16 + ( ( 4 * n + ( c >> 2 ) ) ^ ( 4 * g4 ) ) * 16 + ( c & 3 ) * 4 : tr_at ^ ( 32 * n ) );
  }
  // buffer: 0 or 1, j % 2
  auto stage = [&]( uint32_t j, auto buffer ) __attribute__( ( always_inline ) ) {
    constexpr uint32_t B = decltype( buffer )::value, K0 = B * TILE, K1 = K0 + TILE / 2, V0 = ( 2 + B ) * TILE, V1 = V0 + TILE / 2;
    uint4* const kt = tiles[B];
    uint4* const vt = tiles[2 + B];
    Chunk kf[NU][KK];
    read_keys<CH, K0, K1>( k_lds, kf ); // all but the 2 NU IPG loads of stage j + 1 have landed
    __builtin_amdgcn_sched_barrier( 0 );
    describe( j + 2 );
    fetch( kt, k_at ); // the tile has been read
    mfma_f32x4 st[NU];
#pragma unroll
    for ( uint32_t u = 0; u < NU; u++ ) {
      st[u] = mfma_f32x4 { 0, 0, 0, 0 };
#pragma unroll
      for ( uint32_t kk = 0; kk < KK; kk++ ) {
        if constexpr ( F32 ) {
#pragma unroll
          for ( int e = 0; e < 4; e++ ) {
            st[u] = __builtin_amdgcn_mfma_f32_16x16x4f32( kf[u][kk][e], qb[kk][e], st[u], 0, 0, 0 );
          }
        } else {
          st[u] = Mfma<E>::k32( kf[u][kk], qb[kk], st[u] );
        }
      }
    }
    const uint32_t key0 = k_begin + KEYS * ( j * W + wave );
    if ( key0 + KEYS > k_end ) {
#pragma unroll
      for ( uint32_t e = 0; e < 4 * NU; e++ ) {
        st[e >> 2][e & 3] = key0 + 16 * ( e >> 2 ) + 4 * g4 + ( e & 3 ) < k_end ? st[e >> 2][e & 3] : -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for ( uint32_t u = 0; u < NU; u++ ) {
      mx = fmaxf( mx, fmaxf( fmaxf( st[u][0], st[u][1] ), fmaxf( st[u][2], st[u][3] ) ) );
    }
    mx = column_max( mx ) * a.scale_log2e;
    if ( __builtin_amdgcn_ballot_w64( mx > m + LAZY ) != 0 ) {
      const float m_new = fmaxf( m, mx ), alpha = m_new == -INFINITY ? 1.0f : fast_exp2( m - m_new );
      m = m_new;
      l *= alpha;
#pragma unroll
      for ( uint32_t n = 0; n < NB; n++ ) {
        acc[n] *= alpha;
      }
    }
    const float ms = m == -INFINITY ? 0.0f : m - LIFT<E>;
    float p[4 * NU], sum[2] = { 0, 0 };
#pragma unroll
    for ( uint32_t e = 0; e < 4 * NU; e++ ) {
      p[e] = fast_exp2( __builtin_fmaf( st[e >> 2][e & 3], a.scale_log2e, -ms ) );
      sum[e & 1] += rounded<E>( p[e] );
    }
    l += sum[0] + sum[1];
    Values<E, NB, NU> v;
    v.template read<CH, V0, V1>( v_lds );
    __builtin_amdgcn_sched_barrier( 0 );
    fetch( vt, v_at );
    __builtin_amdgcn_sched_barrier( 0 );
    v.add( p, acc );
  };

  if ( n_mine != 0 ) {
    look_up( 0 );
    describe( 0 );
    fetch( tiles[0], k_at );
    fetch( tiles[2], v_at );
    describe( 1 );
    fetch( tiles[1], k_at );
    fetch( tiles[3], v_at );
    for ( uint32_t j = 0; j < n_mine; j += 2 ) { // (loads past the end fetch nothing, so that the count of those on their way stays the same)
      stage( j, std::integral_constant<uint32_t, 0> {} );
      if ( j + 1 < n_mine ) {
        stage( j + 1, std::integral_constant<uint32_t, 1> {} );
      }
    }
  }
  __builtin_amdgcn_s_waitcnt( 0x0F70 ); // vmcnt(0): nothing is on its way to LDS any more
  l = column_sum( l );

  if constexpr ( W > 1 ) {
    // the waves' parts added up by wave 0, lane for lane as they lie in the registers
    constexpr uint32_t PART = 64 * ( 4 * NB + 2 );
    static_assert( ( W - 1 ) * PART * 4 <= sizeof( s_tiles ), "the parts fit" );
    float* parts = reinterpret_cast<float*>( s_tiles );
    __syncthreads();
    if ( wave != 0 ) {
      float* part = parts + ( wave - 1 ) * PART;
      part[lane] = m;
      part[64 + lane] = l;
#pragma unroll
      for ( uint32_t n = 0; n < NB; n++ ) {
#pragma unroll
        for ( int i = 0; i < 4; i++ ) {
          part[( 2 + 4 * n + i ) * 64 + lane] = acc[n][i];
        }
      }
    }
    __syncthreads();
    if ( wave != 0 ) {
      return;
    }
    float mm = m;
#pragma unroll
    for ( int w = 0; w < W - 1; w++ ) {
      mm = fmaxf( mm, parts[w * PART + lane] );
    }
    const float mm_safe = mm == -INFINITY ? 0.0f : mm, w0 = fast_exp2( m - mm_safe );
    m = mm;
    l *= w0;
#pragma unroll
    for ( uint32_t n = 0; n < NB; n++ ) {
      acc[n] *= w0;
    }
#pragma unroll
    for ( int w = 0; w < W - 1; w++ ) {
      const float* part = parts + w * PART;
      const float ww = fast_exp2( part[lane] - mm_safe );
      l = __builtin_fmaf( part[64 + lane], ww, l );
#pragma unroll
      for ( uint32_t n = 0; n < NB; n++ ) {
#pragma unroll
        for ( int i = 0; i < 4; i++ ) {
          acc[n][i] = __builtin_fmaf( part[( 2 + 4 * n + i ) * 64 + lane], ww, acc[n][i] );
        }
      }
    }
  }
  if ( !ok ) {
    return;
  }
  const uint64_t slot = place * a.splits + b.split;
  const float inv = 1.0f / l;
#pragma unroll
  for ( uint32_t n = 0; n < NB; n++ ) {
    const uint32_t d = 16 * n + 4 * g4;
    if ( d < a.size ) {
      if ( a.splits > 1 ) {
        *reinterpret_cast<mfma_f32x4*>( a.part_out + slot * a.size + d ) = acc[n];
      } else {
        store4( out + place * a.size + d, acc[n][0] * inv, acc[n][1] * inv, acc[n][2] * inv, acc[n][3] * inv );
      }
    }
  }
  if ( a.splits > 1 && g4 == 0 ) {
    a.part_ml[slot * 2] = m - LIFT<E>;
    a.part_ml[slot * 2 + 1] = l;
  }
}

template<typename E, int CH, int W, int HW>
__global__ __launch_bounds__( 64 * W * HW ) void attn_pages_decode_kernel( const E* __restrict__ q, E* __restrict__ out, Call a )
{
  decode_run<E, CH, W, HW>( q, out, a );
}

// =================================================================================================
// decode in fp32 with one query head a kv head, heads of up to CH chunks of 16 bytes: the same walk, products in the vector ALU
//
// One column leaves 15 of the matrix instruction's 16 idle, at 32 cycles each, and where few contexts make a wave's stages a chain those are what it waits for.
// A lane has chunk lane % CH of rows lane / CH, + 64 / CH, ...: a key's score is 4 products and a sum over CH lanes, its values 4 products of the lane's own dims.
// 16 contexts of 33 to 1023 keys, 12 heads of 64: 16.3 us (3.2 TB/s), in matrix instructions 18.8.  Eight stages a wave, one after the other, are what is left.
// =================================================================================================
// sum over the CH (16 or 32) lanes that share a row, in all of them
template<int CH>
__device__ __forceinline__ float lanes_sum( float v )
{
  v = row16_sum( v );
  return CH == 32 ? sum_rows( v, v ) : v;
}

template<int CH, int W>
__device__ __forceinline__ void decode_run_one( const float* __restrict__ q, float* __restrict__ out, const Call& a )
{
  constexpr uint32_t KEYS = 512 / CH, RPI = 64 / CH, LOADS = KEYS / RPI; // 8 loads for a stage's K, and for its V
  constexpr uint32_t TILE = KEYS * CH * 16;                              // bytes
  static_assert( LOADS == 8 && TILE == 8192, "" );
  __shared__ mfma_f32x4 s_tiles[W][4][KEYS * CH]; // of every wave: K of even and of odd stages, V of even and of odd stages

  const uint32_t wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane( threadIdx.x >> 6 ), lane = threadIdx.x & 63, c = lane % CH, r = lane / CH;
  Block b;
  if ( !block_of<true, 16>( a, blockIdx.x / a.n_kv_heads, blockIdx.x % a.n_kv_heads, blockIdx.y, &b ) ) {
    return;
  }
  const uint32_t length = b.start + 1, k_begin = b.split * a.chunk, k_end = min( length, k_begin + a.chunk );
  if ( k_begin >= k_end ) {
    return;
  }
  const uint64_t place = (uint64_t)b.row0 * a.n_kv_heads + b.h;
  const bool ok = 4 * c < a.size; // the lane's chunk is one of the head's
  const mfma_f32x4 qd = ok ? *reinterpret_cast<const mfma_f32x4*>( q + place * a.size + 4 * c ) : mfma_f32x4 {};
  const uint32_t at = ok ? r * a.pages.row_bytes + 16 * c : 0x80000000u, k_off = b.h * a.size * 4, v_off = ( a.n_kv_heads + b.h ) * a.size * 4;

  const uint32_t n_stages = ( k_end - k_begin + KEYS - 1 ) / KEYS, n_mine = n_stages > wave ? ( n_stages - wave + W - 1 ) / W : 0;
  typedef const uint32_t __attribute__( ( address_space( 4 ) ) ) * scalar_ptr;
  const scalar_ptr table = (scalar_ptr)( reinterpret_cast<uintptr_t>( a.pages.table + (uint64_t)b.seq * a.pages.table_stride ) );
  constexpr uint32_t NU = KEYS / 16;
  uint32_t id[NU];
  auto look_up = [&]( uint32_t stage ) __attribute__( ( always_inline ) ) {
#pragma unroll
    for ( uint32_t u = 0; u < NU; u++ ) {
      id[u] = table[min( k_begin + KEYS * ( stage * W + wave ) + 16 * u, k_end - 1 ) >> a.pages.shift];
    }
  };
  __amdgpu_buffer_rsrc_t rsrc[NU];
  auto describe = [&]( uint32_t stage ) __attribute__( ( always_inline ) ) {
#pragma unroll
    for ( uint32_t u = 0; u < NU; u++ ) {
      const uint32_t key = k_begin + KEYS * ( stage * W + wave ) + 16 * u;
      const char* base = a.pages.pool + min( id[u], a.pages.last ) * a.pages.stride + (uint64_t)( key & ( ( 1u << a.pages.shift ) - 1 ) ) * a.pages.row_bytes;
      const uint32_t rows = key < k_end ? min( k_end - key, 16u ) : 0u;
      rsrc[u] = __builtin_amdgcn_make_buffer_rsrc( const_cast<char*>( base ), 0, (int)( rows * a.pages.row_bytes ), 0x00020000 );
    }
    look_up( stage + 1 );
  };
  auto fetch = [&]( mfma_f32x4* tile, uint32_t off ) __attribute__( ( always_inline ) ) {
#pragma unroll
    for ( uint32_t t = 0; t < LOADS; t++ ) { // rows RPI t + r
      __builtin_amdgcn_raw_ptr_buffer_load_lds( rsrc[RPI * t / 16], (lds_ptr)( tile + RPI * t * CH ), 16, at, RPI * t % 16 * a.pages.row_bytes + off, 0, 2 );
    }
  };
  mfma_f32x4 acc = {}; // dims 4 c .. 4 c + 3, of rows r
  float m = -INFINITY, l = 0.0f; // m: of the wave; l: of rows r
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_ptr)&s_tiles[wave][0][0] + 16 * lane;
  auto stage = [&]( uint32_t j, auto buffer ) __attribute__( ( always_inline ) ) {
    constexpr uint32_t B = decltype( buffer )::value;
    mfma_f32x4 k[8], v[8];
    read_rows<B * TILE, true>( lds, k ); // all but the 16 loads of stage j + 1 have landed
    __builtin_amdgcn_sched_barrier( 0 );
    describe( j + 2 );
    fetch( s_tiles[wave][B], k_off );
    const uint32_t key0 = k_begin + KEYS * ( j * W + wave );
    float s[8], mx = -INFINITY;
#pragma unroll
    for ( uint32_t t = 0; t < 8; t++ ) {
      s[t] = lanes_sum<CH>( __builtin_fmaf( k[t][0], qd[0], k[t][1] * qd[1] ) + __builtin_fmaf( k[t][2], qd[2], k[t][3] * qd[3] ) );
      s[t] = key0 + RPI * t + r < k_end ? s[t] * a.scale_log2e : -INFINITY;
      mx = fmaxf( mx, s[t] );
    }
    mx = wave_max( mx );
    if ( mx > m + LAZY ) { // the whole wave
      const float alpha = fast_exp2( m - mx );
      m = mx;
      l *= alpha;
      acc *= alpha;
    }
    const float ms = m == -INFINITY ? 0.0f : m;
    read_rows<( 2 + B ) * TILE, false>( lds, v );
    __builtin_amdgcn_sched_barrier( 0 );
    fetch( s_tiles[wave][2 + B], v_off );
#pragma unroll
    for ( uint32_t t = 0; t < 8; t++ ) {
      const float p = fast_exp2( s[t] - ms );
      l += p;
#pragma unroll
      for ( int e = 0; e < 4; e++ ) {
        acc[e] = __builtin_fmaf( p, v[t][e], acc[e] );
      }
    }
  };
  if ( n_mine != 0 ) {
    look_up( 0 );
    describe( 0 );
    fetch( s_tiles[wave][0], k_off );
    fetch( s_tiles[wave][2], v_off );
    describe( 1 );
    fetch( s_tiles[wave][1], k_off );
    fetch( s_tiles[wave][3], v_off );
    for ( uint32_t j = 0; j < n_mine; j += 2 ) { // (loads past the end fetch nothing, so that the count of those on their way stays the same)
      stage( j, std::integral_constant<uint32_t, 0> {} );
      if ( j + 1 < n_mine ) {
        stage( j + 1, std::integral_constant<uint32_t, 1> {} );
      }
    }
  }
  __builtin_amdgcn_s_waitcnt( 0x0F70 ); // vmcnt(0): nothing is on its way to LDS any more
  // the rows r added up, into all lanes
  auto rows_sum = [&]( float x ) { return CH == 16 ? column_sum( x ) : sum_halves( x, x ); };
  l = rows_sum( l );
#pragma unroll
  for ( int e = 0; e < 4; e++ ) {
    acc[e] = rows_sum( acc[e] );
  }
  if constexpr ( W > 1 ) { // and the waves, by wave 0
    mfma_f32x4* parts = &s_tiles[0][0][0];
    float* ml = reinterpret_cast<float*>( parts + W * CH );
    __syncthreads();
    if ( r == 0 ) {
      parts[wave * CH + c] = acc;
    }
    if ( lane == 0 ) {
      ml[2 * wave] = m;
      ml[2 * wave + 1] = l;
    }
    __syncthreads();
    if ( wave != 0 ) {
      return;
    }
    float mm = m;
#pragma unroll
    for ( int w = 1; w < W; w++ ) {
      mm = fmaxf( mm, ml[2 * w] );
    }
    const float mm_safe = mm == -INFINITY ? 0.0f : mm, w0 = fast_exp2( m - mm_safe );
    m = mm;
    l *= w0;
    acc *= w0;
#pragma unroll
    for ( int w = 1; w < W; w++ ) {
      const float ww = fast_exp2( ml[2 * w] - mm_safe );
      l = __builtin_fmaf( ml[2 * w + 1], ww, l );
      const mfma_f32x4 other = parts[w * CH + c];
#pragma unroll
      for ( int e = 0; e < 4; e++ ) {
        acc[e] = __builtin_fmaf( other[e], ww, acc[e] );
      }
    }
  }
  if ( r != 0 || !ok ) {
    return;
  }
  const uint64_t slot = place * a.splits + b.split;
  if ( a.splits > 1 ) {
    *reinterpret_cast<mfma_f32x4*>( a.part_out + slot * a.size + 4 * c ) = acc;
    if ( lane == 0 ) {
      a.part_ml[slot * 2] = m;
      a.part_ml[slot * 2 + 1] = l;
    }
  } else {
    const float inv = 1.0f / l;
    store4( out + place * a.size + 4 * c, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv );
  }
}

template<int CH, int W>
__global__ __launch_bounds__( 64 * W ) void attn_pages_decode_one_kernel( const float* __restrict__ q, float* __restrict__ out, Call a )
{
  decode_run_one<CH, W>( q, out, a );
}

// =================================================================================================
// packed prompts, 16-bit heads of 8 CH elements and fewer: 128 columns a work-group, 32 a wave, stages of 64 keys
//
// Bound by the matrix units where sequences are long.  K and V rows go from memory straight to LDS, two stages of each; a wave fetches 16 rows of a stage, which
// lie in one page, and rows behind the last key of the work-group, like chunks behind a smaller head, lie outside the descriptor and arrive as zeros.
//   S^T = K Q^T     32 x 32 x 16, the queries in registers: a lane gets 16 of 32 keys for its own column, the lane 32 further on the others
//   O^T += V^T P^T  32 x 32 x 16: the weights as they lie are the second operand, the first comes out of LDS with transposing reads
// A wave's stage: the softmax of the stage's scores in the vector ALU, then pairs of (one step of O^T, one step of the NEXT stage's S^T), their LDS operands asked
// for four pairs ahead and the second half of the exponentials computed beside the first pairs.
// The weights are rounded to the storage type for the second product, as the matrix units take them; the sum takes them rounded too.
// Blocks come longest first; where the kv heads are a multiple of 8 the blocks of a head go to one XCD, whose L2 then fetches its rows once.
// (What the rounding leaves would be a second product, half as many matrix instructions again where they bound the kernel.)
// A prompt of 4096 tokens, 8 kv heads of 128 with 8 queries each, f16: 276 to 303 us on the cards seen (0.91 to 1.0 PFLOP/s; by counters the matrix units are busy half the
// time, the vector ALU 0.3 of it, LDS reads a quarter, which do not overlap fully with two waves a SIMD).  9 prompts of 1 to 1023 tokens behind 0 to 1500 keys, 32 heads, bf16:
// 97 us (0.62; matrix units 0.29): a work-group begins with some 6 us of dependent loads, and the last ones have a CU to themselves.
// =================================================================================================
typedef _Float16 f16x2 __attribute__( ( ext_vector_type( 2 ) ) );
typedef __bf16 b16x2 __attribute__( ( ext_vector_type( 2 ) ) );

// sum + the two weights of a packed pair
template<typename E>
__device__ __forceinline__ float add_pair( uint32_t pair, float sum )
{
  if constexpr ( std::is_same_v<E, __half> ) {
    return __builtin_amdgcn_fdot2( __builtin_bit_cast( f16x2, pair ), f16x2 { (_Float16)1.0f, (_Float16)1.0f }, sum, false );
  } else {
    return __builtin_amdgcn_fdot2_f32_bf16( __builtin_bit_cast( b16x2, pair ), b16x2 { (__bf16)1.0f, (__bf16)1.0f }, sum, false );
  }
}

template<typename E, int CH>
__device__ __forceinline__ void packed_run( const E* __restrict__ q, E* __restrict__ out, const Call& a )
{
  constexpr uint32_t RPI = 64 / CH, IPG = 16 / RPI;          // rows of a load, loads for the wave's 16 rows
  constexpr int SK = CH / 2, I4 = CH / 4, NP = 4 * I4;       // steps of 16 dims of the scores; blocks of 32 dims; pairs of steps of a stage
  using X8 = typename Mfma<E>::x8;
  __shared__ uint4 s_k0[64 * CH], s_k1[64 * CH], s_v0[64 * CH], s_v1[64 * CH]; // named apart: the loop below says at compile time which one it works on

  const uint32_t wave = __builtin_amdgcn_readfirstlane( threadIdx.x >> 6 ), lane = threadIdx.x & 63, r = lane & 31, g2 = lane >> 5;
  uint32_t number, h;
  number_and_head( a, &number, &h );
  Block b;
  if ( !block_of<false, 128>( a, number, h, blockIdx.y, &b ) ) {
    return;
  }
  const uint32_t n_heads = a.n_kv_heads * a.gqa, n_cols = b.tokens * a.gqa;
  const uint32_t k_begin = b.split * a.chunk, k_most = k_begin + a.chunk;
  auto end_of = [&]( uint32_t token ) { return min( visible( a, b, token ), k_most ); }; // keys a token attends of this split: [k_begin, end)
  const uint32_t wg_end = __builtin_amdgcn_readfirstlane( end_of( ( min( n_cols, b.col0 + 128 ) - 1 ) / a.gqa ) );
  if ( wg_end <= k_begin ) {
    return;
  }
  const uint32_t first_col = b.col0 + 32 * wave;
  const bool wave_ok = first_col < n_cols; // a wave without columns still fetches its share of every stage
  const uint32_t t_end = __builtin_amdgcn_readfirstlane( wave_ok ? end_of( ( min( n_cols, first_col + 32 ) - 1 ) / a.gqa ) : 0 ); // of some column of the wave
  const uint32_t t_all = __builtin_amdgcn_readfirstlane( wave_ok ? end_of( first_col / a.gqa ) : 0 );                               // of every column
  const uint32_t col = first_col + r;
  const bool ok = col < n_cols;
  const uint32_t token = ok ? col / a.gqa : 0, head = h * a.gqa + ( ok ? col % a.gqa : 0 );
  const uint32_t my_end = ok ? end_of( token ) : 0;
  const uint64_t place = (uint64_t)( b.row0 + token ) * n_heads + head;

  X8 qb[SK];
#pragma unroll
  for ( int s = 0; s < SK; s++ ) {
    const uint32_t d = 8 * ( 2 * s + g2 );
    qb[s] = ok && d < a.size ? *reinterpret_cast<const X8*>( q + place * a.size + d ) : X8 { 0, 0, 0, 0, 0, 0, 0, 0 };
  }

  mfma_f32x16 acc[I4]; // element v of acc[i]: dim 32 i + 8 (v / 4) + 4 g2 + v % 4 of the lane's column
#pragma unroll
  for ( int i = 0; i < I4; i++ ) {
#pragma unroll
    for ( int v = 0; v < 16; v++ ) {
      acc[i][v] = 0.0f;
    }
  }
  float m = -INFINITY, l = 0.0f; // m: within LAZY of the column's maximum; l: this lane's share

  // a lane's place in the rows of a load; chunks behind the head far outside every descriptor
  const uint32_t ld_row = lane / CH, ld_slot = lane % CH, chunks = a.size / 8;
  const uint32_t k_off = h * a.size * 2, v_off = ( a.n_kv_heads + h ) * a.size * 2;
  auto k_swizzle = []( uint32_t row ) { return CH >= 16 ? row & 15 : ( row >> 1 ) & 7; };
  auto v_swizzle = []( uint32_t row ) { return CH >= 16 ? 4 * ( row & 3 ) : 4 * ( ( row >> 1 ) & 1 ); };
  uint32_t k_at[IPG], v_at[IPG];
#pragma unroll
  for ( uint32_t t = 0; t < IPG; t++ ) {
    const uint32_t row = RPI * t + ld_row, kc = ld_slot ^ k_swizzle( row ), vc = ld_slot ^ v_swizzle( row );
    k_at[t] = kc < chunks ? row * a.pages.row_bytes + k_off + 16 * kc : 0x80000000u;
    v_at[t] = vc < chunks ? row * a.pages.row_bytes + v_off + 16 * vc : 0x80000000u;
  }
  // page numbers by scalar loads, a stage before they are needed
  typedef const uint32_t __attribute__( ( address_space( 4 ) ) ) * scalar_ptr;
  const scalar_ptr table = (scalar_ptr)( reinterpret_cast<uintptr_t>( a.pages.table + (uint64_t)b.seq * a.pages.table_stride ) );
  auto look_up = [&]( uint32_t stage ) __attribute__( ( always_inline ) ) { return table[min( k_begin + 64 * stage + 16 * wave, wg_end - 1 ) >> a.pages.shift]; };
  auto describe = [&]( uint32_t stage, uint32_t id ) __attribute__( ( always_inline ) ) {
    const uint32_t key = k_begin + 64 * stage + 16 * wave;
    const char* base = a.pages.pool + min( id, a.pages.last ) * a.pages.stride + (uint64_t)( key & ( ( 1u << a.pages.shift ) - 1 ) ) * a.pages.row_bytes;
    const uint32_t rows = key < wg_end ? min( wg_end - key, 16u ) : 0u;
    return __builtin_amdgcn_make_buffer_rsrc( const_cast<char*>( base ), 0, (int)( rows * a.pages.row_bytes ), 0x00020000 );
  };
  auto fetch = [&]( __amdgpu_buffer_rsrc_t rsrc, uint4* tile, const uint32_t( &at )[IPG] ) __attribute__( ( always_inline ) ) {
#pragma unroll
    for ( uint32_t t = 0; t < IPG; t++ ) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds( rsrc, (lds_ptr)( tile + ( 16 * wave + RPI * t ) * CH ), 16, at[t], 0, 0, 0 );
    }
  };

  // transposing reads of V: lane 4 e + p of 16 points at key slot e of its half-wave, dims 16 grp + 4 p .. + 3 of dim block 0
  const uint32_t tr_e = ( lane & 15 ) >> 2, tr_p = lane & 3, tr_grp = ( lane >> 4 ) & 1;
  const uint32_t v_lane = ( 4 * g2 + tr_e ) * CH * 16 + ( ( ( 2 * tr_grp + ( tr_p >> 1 ) ) ^ v_swizzle( 4 * g2 + tr_e ) ) * 16 ) + ( tr_p & 1 ) * 8;

  X8 ka[4];
  auto read_k = [&]( const uint4* kt, int n ) __attribute__( ( always_inline ) ) {
    const uint32_t row = 32 * ( n / SK ) + r;
    ka[n & 3] = __builtin_bit_cast( X8, kt[row * CH + ( ( 2 * ( n % SK ) + g2 ) ^ k_swizzle( r ) )] );
  };
  auto score_step = [&]( mfma_f32x16( &st )[2], int n ) __attribute__( ( always_inline ) ) {
    if ( n % SK == 0 ) {
      const mfma_f32x16 zero = { 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0 };
      st[n / SK] = Mfma<E>::k16( ka[n & 3], qb[n % SK], zero );
    } else {
      st[n / SK] = Mfma<E>::k16( ka[n & 3], qb[n % SK], st[n / SK] );
    }
  };
  v4s va[4][2];
  auto read_v = [&]( const uint4* vt, int n ) __attribute__( ( always_inline ) ) {
#pragma unroll
    for ( int half = 0; half < 2; half++ ) {
      va[n & 3][half] = __builtin_amdgcn_ds_read_tr16_b64_v4i16( (lds_v4s)( (lds_char*)vt + ( v_lane ^ ( 64 * ( n % I4 ) ) ) + ( 16 * ( n / I4 ) + 8 * half ) * CH * 16 ) );
    }
  };

  // Behind the barrier of stage i every wave is done with K of stage i (whose scores were made in stage i - 1) and with V of stage i - 1, so K of stage i + 2
  // and V of stage i + 1 are asked for into their places; the barrier of stage i + 1 waits for them.
  const uint32_t n_stages = ( wg_end - k_begin + 63 ) / 64, my_stages = t_end > k_begin ? ( t_end - k_begin + 63 ) / 64 : 0;
  __amdgpu_buffer_rsrc_t next = describe( 0, look_up( 0 ) );
  fetch( next, s_k0, k_at );
  fetch( next, s_v0, v_at );
  next = describe( 1, look_up( 1 ) ); // of stage i + 1
  fetch( next, s_k1, k_at );
  uint32_t id = look_up( 2 ); // of stage i + 2
  // the first stage's keys have landed; its values and the second's keys (2 IPG loads) are waited for at the top of the loop
  __builtin_amdgcn_s_waitcnt( CH == 32 ? 0x4F70 : CH == 16 ? 0x0F78 : 0x0F74 );
  __syncthreads();
  mfma_f32x16 st_a[2], st_b[2]; // scores of even and of odd stages
  if ( my_stages > 0 ) {
#pragma unroll
    for ( int n = 0; n < 4; n++ ) {
      read_k( s_k0, n );
    }
#pragma unroll
    for ( int n = 0; n < NP; n++ ) {
      score_step( st_a, n );
      if ( n + 4 < NP ) {
        read_k( s_k0, n + 4 );
      }
    }
  }

  auto stage = [&]( uint32_t i, uint4* k_cur, uint4* v_cur, uint4* k_nxt, uint4* v_nxt, mfma_f32x16( &st )[2], mfma_f32x16( &st_nxt )[2] ) __attribute__( ( always_inline ) ) {
    const uint32_t t0 = k_begin + 64 * i;
    __builtin_amdgcn_s_waitcnt( 0x0F70 ); // vmcnt(0): what this wave asked for has landed, behind the barrier what all did
    __syncthreads();
    if ( i + 1 < n_stages ) {
      fetch( next, v_nxt, v_at );
    }
    if ( i + 2 < n_stages ) {
      next = describe( i + 2, id );
      fetch( next, k_cur, k_at );
      id = look_up( i + 3 );
    }
    if ( i >= my_stages ) {
      return; // the whole wave
    }
#pragma unroll
    for ( int n = 0; n < 4; n++ ) { // the softmax gives them the time to arrive
      read_v( v_cur, n );
      read_k( k_nxt, n );
    }
    __builtin_amdgcn_sched_barrier( 0 );
    if ( __builtin_amdgcn_readfirstlane( t0 + 64 > t_all ) ) { // keys that some column does not see
      asm volatile( "" ::: "memory" ); // keeps this a branch: the selects are only paid for here
#pragma unroll
      for ( int sub = 0; sub < 2; sub++ ) {
#pragma unroll
        for ( int v = 0; v < 16; v++ ) {
          st[sub][v] = t0 + 32 * sub + 8 * ( v / 4 ) + 4 * g2 + ( v % 4 ) < my_end ? st[sub][v] : -INFINITY;
        }
      }
    }
    float m4[4]; // independent chains
#pragma unroll
    for ( int c = 0; c < 4; c++ ) {
      m4[c] = st[c >> 1][8 * ( c & 1 )];
#pragma unroll
      for ( int e = 1; e < 8; e++ ) {
        m4[c] = fmaxf( m4[c], st[c >> 1][8 * ( c & 1 ) + e] );
      }
    }
    const float mx = half_wave_max( fmaxf( fmaxf( m4[0], m4[1] ), fmaxf( m4[2], m4[3] ) ) ) * a.scale_log2e;
    if ( __builtin_amdgcn_ballot_w64( mx > m + LAZY ) != 0 ) {
      const float m_new = fmaxf( m, mx ), alpha = m_new == -INFINITY ? 1.0f : fast_exp2( m - m_new );
      m = m_new;
      l *= alpha;
#pragma unroll
      for ( int i4 = 0; i4 < I4; i4++ ) {
#pragma unroll
        for ( int v = 0; v < 16; v++ ) {
          acc[i4][v] *= alpha;
        }
      }
    }
    const float ms = m == -INFINITY ? 0.0f : m - LIFT<E>;
    // weights of keys 16 kk .. 16 kk + 15, packed as the second operand of their steps
    typedef uint32_t u32x4 __attribute__( ( ext_vector_type( 4 ) ) );
    u32x4 pk[4];
    float sum[2] = { 0.0f, 0.0f };
    auto weights = [&]( int kk, int e0 ) __attribute__( ( always_inline ) ) {
      float p[2];
#pragma unroll
      for ( int e = 0; e < 2; e++ ) {
        p[e] = fast_exp2( st[kk >> 1][8 * ( kk & 1 ) + e0 + e] * a.scale_log2e - ms );
      }
      const uint32_t pair = rounded_pair<E>( p[0], p[1] );
      sum[( e0 >> 1 ) & 1] = add_pair<E>( pair, sum[( e0 >> 1 ) & 1] );
      pk[kk][e0 >> 1] = pair;
    };
#pragma unroll
    for ( int kk = 0; kk < 2; kk++ ) {
#pragma unroll
      for ( int e0 = 0; e0 < 8; e0 += 2 ) {
        weights( kk, e0 );
      }
    }
    __builtin_amdgcn_s_setprio( 1 ); // before the other wave of the SIMD while this one has matrix work: their softmaxes fall beside it (4096 tokens: 300 us, so 295)
    __builtin_amdgcn_sched_barrier( 0 );
#pragma unroll
    for ( int n = 0; n < NP; n++ ) {
      const int kk = n / I4, i4 = n % I4;
      const v4s lo = va[n & 3][0], hi = va[n & 3][1];
      acc[i4] = Mfma<E>::k16( __builtin_bit_cast( X8, ( v8s { lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3] } ) ), __builtin_bit_cast( X8, pk[kk] ), acc[i4] );
      score_step( st_nxt, n ); // (behind the wave's last stage nothing uses them)
      if ( n + 4 < NP ) {
        read_v( v_cur, n + 4 );
        read_k( k_nxt, n + 4 );
      }
      if ( n < NP / 2 ) { // vector ALU work beside the matrix units
#pragma unroll
        for ( int e0 = ( 8 * i4 / I4 + 1 ) / 2 * 2; e0 < 8 * ( i4 + 1 ) / I4; e0 += 2 ) { // the pair, pairs or half of the steps a pair
          weights( 2 + kk, e0 );
        }
      }
      __builtin_amdgcn_sched_barrier( 0 );
    }
    __builtin_amdgcn_s_setprio( 0 );
    l += sum[0] + sum[1];
  };
  for ( uint32_t i = 0; i < n_stages; i += 2 ) {
    stage( i, s_k0, s_v0, s_k1, s_v1, st_a, st_b );
    if ( i + 1 < n_stages ) {
      stage( i + 1, s_k1, s_v1, s_k0, s_v0, st_b, st_a );
    }
  }

  l += __shfl_xor( l, 32, WAVE );
  float probe = 0.0f;
#pragma unroll
  for ( int i = 0; i < I4; i++ ) {
#pragma unroll
    for ( int v = 0; v < 16; v++ ) {
      probe += 0.0f * acc[i][v];
    }
  }
  const bool mine = ok && k_begin < my_end;
  const uint64_t bad = __builtin_amdgcn_ballot_w64( mine && probe != probe && l == l );
  const uint32_t again = (uint32_t)bad | (uint32_t)( bad >> 32 ); // columns
  if ( mine ) {
    if ( a.splits > 1 ) {
      const uint64_t slot = place * a.splits + b.split;
#pragma unroll
      for ( int i = 0; i < I4; i++ ) {
#pragma unroll
        for ( int v = 0; v < 16; v += 4 ) {
          const uint32_t d = 32 * i + 2 * v + 4 * g2;
          if ( d < a.size ) {
            *reinterpret_cast<float4*>( a.part_out + slot * a.size + d ) = make_float4( acc[i][v], acc[i][v + 1], acc[i][v + 2], acc[i][v + 3] );
          }
        }
      }
      if ( g2 == 0 ) {
        a.part_ml[slot * 2] = m - LIFT<E>;
        a.part_ml[slot * 2 + 1] = l;
      }
    } else {
      const float inv = 1.0f / l;
#pragma unroll
      for ( int i = 0; i < I4; i++ ) {
#pragma unroll
        for ( int v = 0; v < 16; v += 4 ) {
          const uint32_t d = 32 * i + 2 * v + 4 * g2;
          if ( d < a.size ) {
            *reinterpret_cast<uint2*>( out + place * a.size + d )
              = make_uint2( rounded_pair<E>( acc[i][v] * inv, acc[i][v + 1] * inv ), rounded_pair<E>( acc[i][v + 2] * inv, acc[i][v + 3] * inv ) );
          }
        }
      }
    }
  }
  if ( again != 0 ) {
    masked_again<E, CH / 2, true, 1>( q, out, a, b, first_col, again, k_begin, k_most, t_all, wg_end );
  }
}

template<typename E, int CH>
__global__ __launch_bounds__( 256, CH == 32 ? 1 : 2 ) void attn_pages_packed_kernel( const E* __restrict__ q, E* __restrict__ out, Call a )
{
  packed_run<E, CH>( q, out, a );
}

// =================================================================================================
// packed prompts in fp32, heads of up to CH chunks of 16 bytes: 16 CG columns a work-group of two times CG waves, 16 a wave
//
// Bound by the fp32 matrix instruction (16 x 16, 4 deep) where sequences are long.  Stages of 1024 / CH keys (32 at least), two of them in LDS: K and V rows go there straight from
// memory, the next stage's while one is computed, one barrier a stage; rows behind the last key and chunks behind a smaller head arrive as zeros.
// The first CG waves take the first half of every stage's keys, the others the second half for the same columns, and are joined through LDS at the end: the longest
// block of a launch is what a launch of few waits for.
//   S^T = K Q^T     a 16-byte chunk of a key is four steps of the instruction; the scores of a lane: keys 4 g + i of column c
//   O^T += V^T P^T  the weights are the second operand as they lie, V is read value by value: dim c of a block, of keys 4 g + i
// Chunks are swizzled by the row so that both reads touch every bank once.
// 5 prompts of 100 to 900 tokens, 12 heads of 64: 36 us, 70 TFLOP/s; one of 4000, 8 heads of 256: 712 us, 92 TFLOP/s (in the tile kernel above 1992).
// =================================================================================================
template<int CH, int CG>
__device__ __forceinline__ void packed_run_f32( const float* __restrict__ q, float* __restrict__ out, const Call& a )
{
  constexpr uint32_t KEYS = CH == 64 ? 32 : 1024 / CH, TILES = KEYS / 32, RPI = 64 / CH, KK = CH / 4, NB = CH / 4;
  constexpr uint32_t LOADS = KEYS / RPI / ( 2 * CG ); // of a wave for a stage's K, and for its V
  __shared__ mfma_f32x4 s_k0[KEYS * CH], s_k1[KEYS * CH], s_v0[KEYS * CH], s_v1[KEYS * CH];

  const uint32_t loader = __builtin_amdgcn_readfirstlane( threadIdx.x >> 6 ), wave = loader % CG, part = loader / CG, lane = threadIdx.x & 63, c = lane & 15, g4 = lane >> 4;
  uint32_t number, h;
  number_and_head( a, &number, &h );
  Block b;
  if ( !block_of<false, 16 * CG>( a, number, h, blockIdx.y, &b ) ) {
    return;
  }
  const uint32_t n_heads = a.n_kv_heads * a.gqa, n_cols = b.tokens * a.gqa;
  const uint32_t k_begin = b.split * a.chunk, k_most = k_begin + a.chunk;
  auto end_of = [&]( uint32_t token ) { return min( visible( a, b, token ), k_most ); }; // keys a token attends of this split: [k_begin, end)
  const uint32_t wg_end = __builtin_amdgcn_readfirstlane( end_of( ( min( n_cols, b.col0 + 16 * CG ) - 1 ) / a.gqa ) );
  if ( wg_end <= k_begin ) {
    return;
  }
  const uint32_t first_col = b.col0 + 16 * wave;
  const bool wave_ok = first_col < n_cols; // a wave without columns still fetches its share of every stage
  const uint32_t t_end = __builtin_amdgcn_readfirstlane( wave_ok ? end_of( ( min( n_cols, first_col + 16 ) - 1 ) / a.gqa ) : 0 ); // of some column of the wave
  const uint32_t t_all = __builtin_amdgcn_readfirstlane( wave_ok ? end_of( first_col / a.gqa ) : 0 );                               // of every column
  const uint32_t col = first_col + c;
  const bool ok = col < n_cols;
  const uint32_t token = ok ? col / a.gqa : 0, head = h * a.gqa + ( ok ? col % a.gqa : 0 );
  const uint32_t my_end = ok ? end_of( token ) : 0;
  const uint64_t place = (uint64_t)( b.row0 + token ) * n_heads + head;

  mfma_f32x4 qb[KK];
#pragma unroll
  for ( uint32_t kk = 0; kk < KK; kk++ ) {
    const uint32_t d = 4 * ( 4 * kk + g4 );
    qb[kk] = ok && d < a.size ? *reinterpret_cast<const mfma_f32x4*>( q + place * a.size + d ) : mfma_f32x4 {};
  }
  mfma_f32x4 acc[NB]; // element i of acc[n]: dim 16 n + 4 g4 + i of column c
#pragma unroll
  for ( uint32_t n = 0; n < NB; n++ ) {
    acc[n] = mfma_f32x4 {};
  }
  float m = -INFINITY, l = 0.0f; // l: of this lane's keys

  // a lane's place in the rows of a load: the wave's loads are rows RPI (LOADS loader + t) + lane / CH of a stage, which lie in one page
  const uint32_t ld_row = lane / CH, ld_slot = lane % CH, chunks = a.size / 4, run = LOADS * RPI * loader & 15; // run: the wave's first row within its 16
  const uint32_t k_off = h * a.size * 4, v_off = ( a.n_kv_heads + h ) * a.size * 4;
  uint32_t k_at[LOADS], v_at[LOADS];
#pragma unroll
  for ( uint32_t t = 0; t < LOADS; t++ ) {
    const uint32_t row = run + RPI * t + ld_row, kc = ld_slot ^ ( row & 15 ), vc = ld_slot ^ ( row & 12 );
    k_at[t] = kc < chunks ? row * a.pages.row_bytes + k_off + 16 * kc : 0x80000000u;
    v_at[t] = vc < chunks ? row * a.pages.row_bytes + v_off + 16 * vc : 0x80000000u;
  }
  typedef const uint32_t __attribute__( ( address_space( 4 ) ) ) * scalar_ptr;
  const scalar_ptr table = (scalar_ptr)( reinterpret_cast<uintptr_t>( a.pages.table + (uint64_t)b.seq * a.pages.table_stride ) );
  const uint32_t first_row = LOADS * RPI * loader - run; // of the wave's 16 rows within a stage
  auto look_up = [&]( uint32_t stage ) __attribute__( ( always_inline ) ) { return table[min( k_begin + KEYS * stage + first_row, wg_end - 1 ) >> a.pages.shift]; };
  auto fetch = [&]( uint32_t stage, uint32_t id, mfma_f32x4* kt, mfma_f32x4* vt ) __attribute__( ( always_inline ) ) {
    const uint32_t key = k_begin + KEYS * stage + first_row;
    const char* base = a.pages.pool + min( id, a.pages.last ) * a.pages.stride + (uint64_t)( key & ( ( 1u << a.pages.shift ) - 1 ) ) * a.pages.row_bytes;
    const uint32_t rows = key < wg_end ? min( wg_end - key, 16u ) : 0u;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc( const_cast<char*>( base ), 0, (int)( rows * a.pages.row_bytes ), 0x00020000 );
#pragma unroll
    for ( uint32_t t = 0; t < LOADS; t++ ) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds( rsrc, (lds_ptr)( kt + ( LOADS * RPI * loader + RPI * t ) * CH ), 16, k_at[t], 0, 0, 0 );
    }
#pragma unroll
    for ( uint32_t t = 0; t < LOADS; t++ ) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds( rsrc, (lds_ptr)( vt + ( LOADS * RPI * loader + RPI * t ) * CH ), 16, v_at[t], 0, 0, 0 );
    }
  };

  const uint32_t n_stages = ( wg_end - k_begin + KEYS - 1 ) / KEYS;
  fetch( 0, look_up( 0 ), s_k0, s_v0 );
  uint32_t id = look_up( 1 ); // of the stage behind the one that is computed
  auto stage = [&]( uint32_t i, const mfma_f32x4* kt, const mfma_f32x4* vt, mfma_f32x4* k_nxt, mfma_f32x4* v_nxt ) __attribute__( ( always_inline ) ) {
    const uint32_t r0 = 16 * TILES * part, t0 = k_begin + KEYS * i + r0; // the wave's first row of the stage, its key
    __builtin_amdgcn_s_waitcnt( 0x0F70 ); // vmcnt(0): what this wave asked for has landed, behind the barrier what all did, and all are done with the stage before
    __syncthreads();
    if ( i + 1 < n_stages ) {
      fetch( i + 1, id, k_nxt, v_nxt );
      id = look_up( i + 2 );
    }
    if ( t0 >= t_end ) {
      return; // the whole wave
    }
    mfma_f32x4 st[TILES];
#pragma unroll
    for ( uint32_t u = 0; u < TILES; u++ ) {
      st[u] = mfma_f32x4 {};
#pragma unroll
      for ( uint32_t kk = 0; kk < KK; kk++ ) {
        const mfma_f32x4 k = kt[( r0 + 16 * u + c ) * CH + ( ( 4 * kk + g4 ) ^ c )];
#pragma unroll
        for ( int e = 0; e < 4; e++ ) {
          st[u] = __builtin_amdgcn_mfma_f32_16x16x4f32( k[e], qb[kk][e], st[u], 0, 0, 0 );
        }
      }
    }
    if ( __builtin_amdgcn_readfirstlane( t0 + 16 * TILES > t_all ) ) { // keys that some column does not see
#pragma unroll
      for ( uint32_t e = 0; e < 4 * TILES; e++ ) {
        st[e >> 2][e & 3] = t0 + 16 * ( e >> 2 ) + 4 * g4 + ( e & 3 ) < my_end ? st[e >> 2][e & 3] : -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for ( uint32_t u = 0; u < TILES; u++ ) {
      mx = fmaxf( mx, fmaxf( fmaxf( st[u][0], st[u][1] ), fmaxf( st[u][2], st[u][3] ) ) );
    }
    mx = column_max( mx ) * a.scale_log2e;
    if ( __builtin_amdgcn_ballot_w64( mx > m + LAZY ) != 0 ) {
      const float m_new = fmaxf( m, mx ), alpha = m_new == -INFINITY ? 1.0f : fast_exp2( m - m_new );
      m = m_new;
      l *= alpha;
#pragma unroll
      for ( uint32_t n = 0; n < NB; n++ ) {
        acc[n] *= alpha;
      }
    }
    const float ms = m == -INFINITY ? 0.0f : m;
    float sum[2] = { 0, 0 };
#pragma unroll
    for ( uint32_t e = 0; e < 4 * TILES; e++ ) {
      st[e >> 2][e & 3] = fast_exp2( __builtin_fmaf( st[e >> 2][e & 3], a.scale_log2e, -ms ) );
      sum[e & 1] += st[e >> 2][e & 3];
    }
    l += sum[0] + sum[1];
    const float* v = reinterpret_cast<const float*>( vt );
#pragma unroll
    for ( uint32_t u = 0; u < TILES; u++ ) {
#pragma unroll
      for ( uint32_t i4 = 0; i4 < 4; i4++ ) {
#pragma unroll
        for ( uint32_t n = 0; n < NB; n++ ) {
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32( v[( r0 + 16 * u + 4 * g4 + i4 ) * CH * 4 + ( ( 4 * n + ( c >> 2 ) ) ^ ( 4 * g4 ) ) * 4 + ( c & 3 )], st[u][i4], acc[n], 0, 0, 0 );
        }
      }
    }
  };
  for ( uint32_t i = 0; i < n_stages; i += 2 ) {
    stage( i, s_k0, s_v0, s_k1, s_v1 );
    if ( i + 1 < n_stages ) {
      stage( i + 1, s_k1, s_v1, s_k0, s_v0 );
    }
  }

  l = column_sum( l );
  // the second half's parts, lane for lane as they lie in the registers
  constexpr uint32_t PART = 64 * ( 4 * NB + 2 );
  static_assert( PART * 4 <= sizeof( s_k0 ), "a wave's part fits one of the arrays" );
  float* parts = reinterpret_cast<float*>( wave == 0 ? s_k0 : wave == 1 ? s_k1 : wave == 2 ? s_v0 : s_v1 );
  __syncthreads();
  if ( part == 1 ) {
    parts[lane] = m;
    parts[64 + lane] = l;
#pragma unroll
    for ( uint32_t n = 0; n < NB; n++ ) {
#pragma unroll
      for ( int i = 0; i < 4; i++ ) {
        parts[( 2 + 4 * n + i ) * 64 + lane] = acc[n][i];
      }
    }
  }
  __syncthreads();
  if ( part == 1 ) {
    return;
  }
  {
    const float other = parts[lane], mm = fmaxf( m, other ), mm_safe = mm == -INFINITY ? 0.0f : mm;
    const float w0 = fast_exp2( m - mm_safe ), w1 = fast_exp2( other - mm_safe );
    m = mm;
    l = l * w0 + parts[64 + lane] * w1;
#pragma unroll
    for ( uint32_t n = 0; n < NB; n++ ) {
#pragma unroll
      for ( int i = 0; i < 4; i++ ) {
        acc[n][i] = __builtin_fmaf( parts[( 2 + 4 * n + i ) * 64 + lane], w1, acc[n][i] * w0 );
      }
    }
  }
  float probe = 0.0f;
#pragma unroll
  for ( uint32_t n = 0; n < NB; n++ ) {
    probe += 0.0f * ( ( acc[n][0] + acc[n][1] ) + ( acc[n][2] + acc[n][3] ) );
  }
  const bool mine = ok && k_begin < my_end;
  const uint64_t bad = __builtin_amdgcn_ballot_w64( mine && probe != probe && l == l );
  uint32_t again = (uint32_t)( bad | bad >> 16 | bad >> 32 | bad >> 48 ) & 0xffff; // columns
  // (asked here as well: 4 prompts of 300 tokens, 32 heads of 128 take 45.7 us so, and 49.4 with the one call behind the stores, by how the loop's instructions fall)
  if ( again != 0 && finite_values<float>( a.pages, b.seq, v_off / 4, a.size, max( k_begin, t_all ), wg_end ) ) {
    again = 0;
  }
  if ( mine && !( again >> c & 1 ) ) {
    const uint64_t slot = place * a.splits + b.split;
    const float inv = a.splits > 1 ? 1.0f : 1.0f / l;
    float* to = a.splits > 1 ? a.part_out + slot * a.size : out + place * a.size;
#pragma unroll
    for ( uint32_t n = 0; n < NB; n++ ) {
      const uint32_t d = 16 * n + 4 * g4;
      if ( d < a.size ) {
        store4( to + d, acc[n][0] * inv, acc[n][1] * inv, acc[n][2] * inv, acc[n][3] * inv );
      }
    }
    if ( a.splits > 1 && g4 == 0 ) {
      a.part_ml[slot * 2] = m;
      a.part_ml[slot * 2 + 1] = l;
    }
  }
  if ( again != 0 ) {
    masked_again<float, NB, true, CG>( q, out, a, b, first_col, again, k_begin, k_most, t_all, wg_end );
  }
}

template<int CH, int CG>
__global__ __launch_bounds__( 128 * CG, CH == 64 ? CG / 2 : CG ) void attn_pages_packed_f32_kernel( const float* __restrict__ q, float* __restrict__ out, Call a )
{
  packed_run_f32<CH, CG>( q, out, a );
}

// =================================================================================================
// splits of a row added up: NW waves of a work-group take a (query row, head), every NW-th split each, eight of them asked for at once.  Bound by latency:
// 96 (row, head)s of 8 splits 4.3 to 4.8 us.
// =================================================================================================
template<typename T, bool DECODE, int NW>
__global__ __launch_bounds__( 256 ) void pages_merge_kernel( T* __restrict__ out, Call a, uint32_t rows )
{
  constexpr int PER = 4 / NW; // (row, head)s of a work-group
  __shared__ float s_part[4][256], s_l[4];
  const uint32_t lane = threadIdx.x & 63, n_heads = a.n_kv_heads * a.gqa, wave = __builtin_amdgcn_readfirstlane( threadIdx.x >> 6 ), turn = wave % NW;
  const uint64_t place = (uint64_t)blockIdx.x * PER + wave / NW;
  const uint32_t row = (uint32_t)( place / n_heads );
  uint32_t keys = 0;
  if ( row < rows ) {
    if constexpr ( DECODE ) {
      keys = min( a.lengths[row], a.max_keys );
    } else {
      const uint32_t seq = packed_sequence( a.seqs, row );
      if ( seq < a.seqs.batch && row - a.seqs.begin( seq ) < a.seqs.count( seq ) ) {
        keys = min( a.seqs.begin_pos( seq ) + ( row - a.seqs.begin( seq ) ) + 1, a.max_keys );
      }
    }
  }
  const uint32_t n = ( keys + a.chunk - 1 ) / a.chunk; // at most a.splits, as max_keys is at most splits * chunk
  const float* ml = a.part_ml + place * a.splits * 2;
  const float* part = a.part_out + place * a.splits * a.size;
  float mm = -INFINITY;
  for ( uint32_t s = lane; s < n; s += 64 ) {
    mm = fmaxf( mm, ml[2 * s] );
  }
  mm = wave_max( mm );
  const float mm_safe = mm == -INFINITY ? 0.0f : mm;
  float l = 0.0f, acc[4] = { 0, 0, 0, 0 };
  for ( uint32_t s0 = 0; s0 < n; s0 += 64 * NW ) { // lane <-> split s0 + NW lane + turn
    const uint32_t mine = s0 + NW * lane + turn;
    const float w = mine < n ? fast_exp2( ml[2 * mine] - mm_safe ) : 0.0f;
    l += wave_sum( mine < n ? w * ml[2 * mine + 1] : 0.0f );
    for ( uint32_t k0 = 0; k0 < 64 && s0 + NW * k0 + turn < n; k0 += 8 ) {
      float v[8][4];
#pragma unroll
      for ( uint32_t k = 0; k < 8; k++ ) {
        const uint32_t split = min( s0 + NW * ( k0 + k ) + turn, n - 1 ); // past the end: the last one, whose weight there is 0 (its values may be infinite)
#pragma unroll
        for ( uint32_t u = 0; u < 4; u++ ) {
          v[k][u] = 64 * u + lane < a.size ? part[(uint64_t)split * a.size + 64 * u + lane] : 0.0f;
        }
      }
#pragma unroll
      for ( uint32_t k = 0; k < 8; k++ ) {
        const float wk = lane_value( w, (int)( k0 + k ) );
        const bool there = s0 + NW * ( k0 + k ) + turn < n;
#pragma unroll
        for ( uint32_t u = 0; u < 4; u++ ) {
          acc[u] = there ? __builtin_fmaf( v[k][u], wk, acc[u] ) : acc[u];
        }
      }
    }
  }
  if constexpr ( NW > 1 ) {
#pragma unroll
    for ( uint32_t u = 0; u < 4; u++ ) {
      s_part[wave][64 * u + lane] = acc[u];
    }
    if ( lane == 0 ) {
      s_l[wave] = l;
    }
    __syncthreads();
    if ( turn != 0 ) {
      return;
    }
    for ( uint32_t w = 1; w < NW; w++ ) {
      l += s_l[wave + w];
#pragma unroll
      for ( uint32_t u = 0; u < 4; u++ ) {
        acc[u] += s_part[wave + w][64 * u + lane];
      }
    }
  }
  if ( n == 0 ) {
    return; // a row that attends nothing is left as it is
  }
#pragma unroll
  for ( uint32_t u = 0; u < 4; u++ ) {
    const uint32_t d = 64 * u + lane;
    if ( d < a.size ) {
      out[place * a.size + d] = from_f32<T>( acc[u] / l );
    }
  }
}

// =================================================================================================
// host side
// =================================================================================================
struct Plan
{
  uint32_t blocks, splits, chunk; // blocks: grid x
  uint32_t n_blocks;
  uint32_t waves; // of a work-group; 0: the kernel that takes everything
  uint32_t longest_first;
  uint64_t bytes;
};

// The kernels that stream to LDS take heads made of 16-byte chunks, runs of 16 keys in one page, and everything aligned to 16 bytes.
bool takes_tiles( const gh_shape* s, gh_dtype dt ) { return s->head_size * dtype_size( dt ) % 16 == 0; }

constexpr uint64_t MOST_PARTS = 65536; // of (query row, head, split) that leave partial results

// How a call is cut.  Splits are whole numbers of 64 keys.
Plan plan_call( bool decode, uint64_t batch, uint64_t rows, uint32_t max_keys, const gh_shape* s, gh_dtype dt, bool tiles )
{
  Plan p {};
  uint32_t cols = decode ? 16 : tiles && dt != GH_F32 ? 128 : 64;
  auto blocks_of = [&] { return most_blocks( rows * s->gqa_size, batch, cols ); };
  // fp32: half as many columns a work-group while there are fewer than two and a half a CU, since a launch of few lasts as long as its longest (5 prompts of 100 to 900 tokens, 12
  // heads of 64: 51 us with 64 columns, 40 with 32; 4 of 300, 32 heads of 128: 46 and 49; 16 of 1000, 12 heads of 64: 254 and 294)
  if ( !decode && tiles && dt == GH_F32 && blocks_of() * s->n_kv_heads * 2 < 5ull * (uint64_t)cu_count() ) {
    cols = 32;
  }
  p.n_blocks = decode ? ( s->gqa_size + cols - 1 ) / cols : 0;
  const uint64_t blocks = decode ? batch * p.n_blocks : blocks_of();
  p.blocks = (uint32_t)blocks;
  if ( decode && tiles ) {
    // Microseconds as measured on MI355X.  A stage of 16 KB takes a wave on its own 0.75, the four waves of a work-group 1.5 (fp32 heads above 128: 2.2, the matrix instructions of their 16 keys), and 2.4 where the waves that fit
    // (four a CU, eight of 16-bit heads up to 64) share the memory's rate; a round of work-groups takes 2 to begin and end; a split adds a launch (4) and 8 bytes an element
    // that go out and come back at 3 TB/s.  Where lengths differ the launch ends on the longest runs: a tenth of a wave's stages.
    // Measured, GQA heads (8 of 8 queries) in f16, us: 1 context of 301 keys, 4 waves 7.0, splits of 64 8.8 | 1 x 4096, 4 waves unsplit 39, splits of 64 10.8 |
    // 16 x 500, 4 waves 9.8, one wave 15.1 | 64 x 4096, splits of 2048 167, of 512 185, of 64 261 | 256 x 1000, one wave 162, 4 waves 177
    // 32 heads of one query: 8 x 2000, 4 waves 42, one wave 48 | 3 x 30000, splits of 1024 233, of 128 248, 4 waves unsplit 269
    const uint64_t streams = batch * p.n_blocks * s->n_kv_heads;
    const bool wide = s->head_size > 128; // twice the bytes and the LDS
    const double slots = cu_count() * ( wide ? 2.0 : dt != GH_F32 && s->head_size <= 64 ? 8.0 : 4.0 );
    const uint32_t stage = dt == GH_F32 && s->head_size > 64 ? 16 : 32; // keys
    double best = 0;
    for ( uint32_t waves = 1; waves <= ( wide ? 2 : 4 ); waves += wide ? 1 : 3 ) {
      for ( uint32_t chunk = 64; chunk != 0; chunk = chunk >= max_keys ? 0 : 2 * chunk ) {
        const uint64_t splits = ( max_keys + chunk - 1 ) / chunk;
        if ( splits > 65535 || ( splits > 1 && rows * s->n_heads * splits > MOST_PARTS ) ) {
          continue;
        }
        const double stages = (double)( ( std::min( chunk, max_keys ) + stage * waves - 1 ) / ( stage * waves ) ), load = (double)( streams * splits * waves ) / slots;
        const double alone = dt == GH_F32 && wide ? 2.2 : waves == 1 ? 0.75 : 1.5, full = std::max( alone, 2.4 * std::min( 1.0, load ) );
        double us = stages * std::max( alone, 2.4 * load ) + 0.1 * stages * full + 2.0 * std::max( 1.0, load );
        if ( splits > 1 ) {
          us += 4.0 + (double)( rows * s->n_heads * splits ) * s->head_size * 8 / 3e6;
        }
        if ( p.waves == 0 || us < best ) {
          best = us;
          p.waves = waves;
          p.chunk = chunk;
          p.splits = (uint32_t)splits;
        }
      }
    }
    // contexts in order of length where work-groups wait for others to end and last long enough to pay for the order
    // (64 contexts of 57 to 4096 keys 102 -> 91 us, of 4096 each 164.0 and 164.9; short calls lost 1 to 2 us of 6 to 17)
    p.longest_first = batch > 1 && batch <= 64 && max_keys >= 1024 && (double)( streams * p.splits * p.waves ) > slots;
    p.bytes = p.splits == 1 ? 0 : rows * s->n_heads * p.splits * ( s->head_size + 2 ) * sizeof( float );
    return p;
  }
  // Few rows of many keys: as many splits as cost least.  A stage of 64 keys takes a work-group 1.1 us (2.6 in fp32); a split adds a launch (5) and 8 bytes an element that go
  // out and come back at 2 TB/s.  us, f16, 8 kv heads of 8 queries: 64 tokens behind 4000 keys, unsplit 76, in 6 33, in 16 35 | 16 behind 30000: 502, in 16 50, in 32 45 |
  // 512 tokens: 20, in 2 48.  fp32, 12 heads of 64: 64 tokens behind 2000 keys: 86, in 16 20, in 32 23.
  const uint64_t groups = blocks * s->n_kv_heads;
  uint64_t splits = 1;
  double best = 0;
  for ( uint64_t n = 1; n <= 256 && ( n == 1 || ( rows * s->n_heads * n <= MOST_PARTS && ( n - 1 ) * 64 < max_keys ) ); n += ( n + 1 ) / 2 ) {
    const double stages = (double)( ( ( max_keys + n - 1 ) / n + 63 ) / 64 ), load = (double)( groups * n ) / ( 2.0 * cu_count() );
    const double us = stages * ( dt == GH_F32 ? 2.6 : 1.1 ) * std::max( 1.0, load ) + ( n > 1 ? 5.0 + (double)( rows * s->n_heads * n ) * s->head_size * 8 / 2e6 : 0.0 );
    if ( n == 1 || us < best ) {
      best = us;
      splits = n;
    }
  }
  p.waves = !tiles ? 0 : dt == GH_F32 ? cols / 8 : 4;
  p.chunk = (uint32_t)( ( ( max_keys + splits - 1 ) / splits + 63 ) / 64 * 64 );
  p.splits = ( max_keys + p.chunk - 1 ) / p.chunk;
  p.bytes = p.splits == 1 ? 0 : rows * s->n_heads * p.splits * ( s->head_size + 2 ) * sizeof( float );
  return p;
}

// Bytes that every plan of at most so many rows and keys fits into.
uint64_t most_bytes( uint64_t rows, uint32_t max_keys, const gh_shape* s )
{
  return max_keys <= 64 ? 0 : std::min<uint64_t>( rows * s->n_heads * ( ( (uint64_t)max_keys + 63 ) / 64 ), MOST_PARTS ) * ( s->head_size + 2 ) * sizeof( float );
}

bool shape_ok( const gh_shape* s )
{
  return s != nullptr && s->head_size > 0 && s->head_size <= 256 && s->n_kv_heads > 0 && s->gqa_size > 0 && s->n_kv_heads <= 65535 && s->gqa_size <= 65535
         && (uint64_t)s->n_kv_heads * s->gqa_size == s->n_heads && (uint64_t)s->n_kv_heads * s->head_size == s->kv_dim;
}

template<typename T, bool DECODE>
void launch_f32( const Plan& p, const Call& a, const void* q, void* out, hipStream_t st )
{
  const dim3 grid( p.blocks, a.n_kv_heads, p.splits );
  const T* tq = static_cast<const T*>( q );
  T* to = static_cast<T*>( out );
  if ( a.size <= 64 ) {
    attn_pages_f32_kernel<T, 4, DECODE><<<grid, 256, 0, st>>>( tq, to, a );
  } else if ( a.size <= 128 ) {
    attn_pages_f32_kernel<T, 8, DECODE><<<grid, 256, 0, st>>>( tq, to, a );
  } else {
    attn_pages_f32_kernel<T, 16, DECODE><<<grid, 256, 0, st>>>( tq, to, a );
  }
}

template<typename E>
void launch_decode_tiles( const Plan& p, const Call& a, const void* q, void* out, hipStream_t st )
{
  const E* tq = static_cast<const E*>( q );
  E* to = static_cast<E*>( out );
  if constexpr ( sizeof( E ) == 4 ) {
    if ( a.gqa == 1 && a.size <= 128 ) {
      const dim3 grid( p.blocks * a.n_kv_heads, p.splits );
      if ( a.size <= 64 ) {
        p.waves > 1 ? attn_pages_decode_one_kernel<16, 4><<<grid, 256, 0, st>>>( tq, to, a ) : attn_pages_decode_one_kernel<16, 1><<<grid, 64, 0, st>>>( tq, to, a );
      } else {
        p.waves > 1 ? attn_pages_decode_one_kernel<32, 4><<<grid, 256, 0, st>>>( tq, to, a ) : attn_pages_decode_one_kernel<32, 1><<<grid, 64, 0, st>>>( tq, to, a );
      }
      return;
    }
  }
  auto go = [&]( auto chunks, auto waves, auto heads ) {
    constexpr int CH = decltype( chunks )::value, W = decltype( waves )::value, HW = decltype( heads )::value;
    attn_pages_decode_kernel<E, CH, W, HW><<<dim3( p.blocks * ( a.n_kv_heads / HW ), p.splits ), 64 * W * HW, 0, st>>>( tq, to, a );
  };
  const std::integral_constant<int, 1> one {};
  const std::integral_constant<int, 2> two {};
  const std::integral_constant<int, 4> four {};
  auto sizes = [&]( auto chunks ) {
    if ( p.waves > 1 ) {
      go( chunks, four, one );
    } else if ( a.n_kv_heads % 2 == 0 ) {
      go( chunks, one, two );
    } else {
      go( chunks, one, one );
    }
  };
  constexpr int NARROW = 4 * sizeof( E ); // chunks of 64 elements
  if ( a.size <= 64 ) {
    sizes( std::integral_constant<int, NARROW> {} );
  } else if ( a.size <= 128 ) {
    sizes( std::integral_constant<int, 2 * NARROW> {} );
  } else { // 64 KB of LDS a wave
    if ( p.waves > 1 ) {
      go( std::integral_constant<int, 4 * NARROW> {}, two, one );
    } else {
      go( std::integral_constant<int, 4 * NARROW> {}, one, one );
    }
  }
}

template<typename E>
void launch_packed_tiles( const Plan& p, const Call& a, const void* q, void* out, hipStream_t st )
{
  const dim3 grid( p.blocks * a.n_kv_heads, p.splits );
  if constexpr ( sizeof( E ) == 4 ) {
    const float* tq = static_cast<const float*>( q );
    float* to = static_cast<float*>( out );
    if ( a.size <= 64 ) {
      p.waves == 8 ? attn_pages_packed_f32_kernel<16, 4><<<grid, 512, 0, st>>>( tq, to, a ) : attn_pages_packed_f32_kernel<16, 2><<<grid, 256, 0, st>>>( tq, to, a );
    } else if ( a.size <= 128 ) {
      p.waves == 8 ? attn_pages_packed_f32_kernel<32, 4><<<grid, 512, 0, st>>>( tq, to, a ) : attn_pages_packed_f32_kernel<32, 2><<<grid, 256, 0, st>>>( tq, to, a );
    } else {
      p.waves == 8 ? attn_pages_packed_f32_kernel<64, 4><<<grid, 512, 0, st>>>( tq, to, a ) : attn_pages_packed_f32_kernel<64, 2><<<grid, 256, 0, st>>>( tq, to, a );
    }
  } else if ( a.size <= 64 ) {
    attn_pages_packed_kernel<E, 8><<<grid, 256, 0, st>>>( static_cast<const E*>( q ), static_cast<E*>( out ), a );
  } else if ( a.size <= 128 ) {
    attn_pages_packed_kernel<E, 16><<<grid, 256, 0, st>>>( static_cast<const E*>( q ), static_cast<E*>( out ), a );
  } else {
    attn_pages_packed_kernel<E, 32><<<grid, 256, 0, st>>>( static_cast<const E*>( q ), static_cast<E*>( out ), a );
  }
}

template<typename T, bool DECODE>
int launch( const Plan& p, const Call& a, const void* q, void* out, uint64_t rows, hipStream_t st )
{
  if ( p.waves == 0 ) {
    launch_f32<T, DECODE>( p, a, q, out, st );
  } else if constexpr ( DECODE ) {
    launch_decode_tiles<T>( p, a, q, out, st );
  } else {
    launch_packed_tiles<T>( p, a, q, out, st );
  }
  GH_LAUNCH_CHECK();
  if ( p.splits > 1 ) {
    const uint64_t places = rows * a.n_kv_heads * a.gqa;
    if ( places < 16ull * (uint64_t)cu_count() ) {
      pages_merge_kernel<T, DECODE, 4><<<(unsigned)places, 256, 0, st>>>( static_cast<T*>( out ), a, (uint32_t)rows );
    } else {
      pages_merge_kernel<T, DECODE, 1><<<(unsigned)( ( places + 3 ) / 4 ), 256, 0, st>>>( static_cast<T*>( out ), a, (uint32_t)rows );
    }
    GH_LAUNCH_CHECK();
  }
  return GH_OK;
}

// Both entry points: `rows` query rows of `batch` sequences (decode: one each).
template<bool DECODE>
int attn_pages( const char* op, const void* q, const gh_pages* pages, const uint32_t* lengths, const uint32_t* first, const uint32_t* start, void* xb, uint64_t batch,
                uint64_t rows, uint32_t max_keys, const gh_shape* s, gh_dtype dt, void* workspace, uint64_t workspace_bytes, gh_stream stream )
{
  const bool empty = batch == 0 || rows == 0 || max_keys == 0;
  Call a {};
  if ( !empty ) { // what can be said without a device is said first
    GH_REQUIRE( shape_ok( s ), "%s: unsupported or inconsistent shape", op );
    if ( int rc = check_pages( op, pages, s->kv_dim, dt, &a.pages ) ) {
      return rc;
    }
    GH_REQUIRE( q && xb && ( DECODE ? lengths != nullptr : first != nullptr ), "%s: NULL pointer", op );
    GH_REQUIRE( ( reinterpret_cast<uintptr_t>( q ) | reinterpret_cast<uintptr_t>( xb ) ) % dtype_size( dt ) == 0, "%s: q or xb is not aligned to its elements", op );
    GH_REQUIRE( max_keys <= a.pages.reach(), "%s: %u keys, the table reaches %u", op, max_keys, a.pages.reach() );
    GH_REQUIRE( batch <= 1u << 20 && rows <= 1u << 24 && rows * s->n_heads < 1ull << 31, "%s: too many rows", op );
    GH_REQUIRE( !overlap( q, rows * s->n_heads * s->head_size * dtype_size( dt ), xb, rows * s->n_heads * s->head_size * dtype_size( dt ) ), "%s: xb over q", op );
  }
  if ( int rc = ensure_init() ) {
    return rc;
  }
  if ( empty ) {
    return GH_OK;
  }
  const uint64_t places = reinterpret_cast<uintptr_t>( pages->pool ) | pages->page_stride | reinterpret_cast<uintptr_t>( q ) | reinterpret_cast<uintptr_t>( xb );
  const Plan p = plan_call( DECODE, batch, rows, max_keys, s, dt, takes_tiles( s, dt ) && places % 16 == 0 && pages->page_tokens >= 16 );
  // (a grid has fewer than 2^32 threads; work-groups have up to 512, the merge kernel 64 a row and head)
  GH_REQUIRE( (uint64_t)p.blocks * s->n_kv_heads < 1u << 23 && ( p.splits == 1 || rows * s->n_heads < 1u << 26 ), "%s: too many work-groups", op );
  GH_REQUIRE( p.bytes == 0 || ( workspace != nullptr && reinterpret_cast<uintptr_t>( workspace ) % 16 == 0 ), "%s: a 16-byte aligned workspace is needed", op );
  if ( p.bytes > workspace_bytes ) {
    return fail( GH_ERR_WORKSPACE, "%s: workspace of %llu bytes, %llu are needed", op, (unsigned long long)workspace_bytes, (unsigned long long)p.bytes );
  }
  a.seqs = { first, start, (uint32_t)batch, (uint32_t)rows };
  a.lengths = lengths;
  a.n_kv_heads = s->n_kv_heads;
  a.gqa = s->gqa_size;
  a.size = s->head_size;
  a.max_keys = max_keys;
  a.chunk = p.chunk;
  a.splits = p.splits;
  a.n_blocks = p.n_blocks;
  a.longest_first = p.longest_first;
  a.scale_log2e = LOG2E / sqrtf( (float)s->head_size );
  a.part_out = static_cast<float*>( workspace );
  a.part_ml = a.part_out + rows * s->n_heads * p.splits * s->head_size;
  hipStream_t st = as_stream( stream );
  switch ( dt ) {
    case GH_F16: return launch<__half, DECODE>( p, a, q, xb, rows, st );
    case GH_BF16: return launch<__bf16, DECODE>( p, a, q, xb, rows, st );
    default: return launch<float, DECODE>( p, a, q, xb, rows, st );
  }
}

} // namespace
} // namespace gh

using namespace gh;

extern "C" {

uint64_t gh_attn_decode_paged_workspace( uint64_t batch, uint32_t max_length, const gh_shape* shape, gh_dtype dt )
{
  return !shape_ok( shape ) || batch == 0 || batch > 1u << 24 ? 0 : most_bytes( batch, max_length, shape );
}

int gh_attn_decode_paged( const void* q, const gh_pages* pages, const uint32_t* lengths_dev, void* xb, uint64_t batch, uint32_t max_length, const gh_shape* shape,
                          gh_dtype dt, void* workspace, uint64_t workspace_bytes, gh_stream stream )
{
  return attn_pages<true>( "gh_attn_decode_paged", q, pages, lengths_dev, nullptr, nullptr, xb, batch, batch, max_length, shape, dt, workspace, workspace_bytes, stream );
}

uint64_t gh_attn_packed_workspace( uint64_t batch, uint64_t n_tokens, uint32_t max_keys, const gh_shape* shape, gh_dtype dt )
{
  return !shape_ok( shape ) || batch == 0 || n_tokens > 1u << 24 ? 0 : most_bytes( n_tokens, max_keys, shape );
}

int gh_attn_packed( const void* q, const gh_pages* pages, const uint32_t* first_dev, const uint32_t* start_pos_dev, void* xb, uint64_t batch, uint64_t n_tokens,
                    uint32_t max_keys, const gh_shape* shape, gh_dtype dt, void* workspace, uint64_t workspace_bytes, gh_stream stream )
{
  return attn_pages<false>( "gh_attn_packed", q, pages, nullptr, first_dev, start_pos_dev, xb, batch, n_tokens, max_keys, shape, dt, workspace, workspace_bytes, stream );
}

} // extern "C"
