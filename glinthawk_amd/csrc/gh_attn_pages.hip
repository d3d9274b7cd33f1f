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
    b->seq = number / a.n_blocks;
    b->col0 = number % a.n_blocks * COLS;
    const uint32_t length = min( a.lengths[b->seq], a.max_keys );
    if ( length == 0 ) {
      return false;
    }
    b->row0 = b->seq;
    b->tokens = 1;
    b->start = length - 1;
    return true;
  } else {
    uint32_t block;
    if ( !packed_block( a.seqs, a.gqa, COLS, number, &b->seq, &block ) ) {
      return false;
    }
    b->col0 = block * COLS;
    b->row0 = a.seqs.begin( b->seq );
    b->tokens = a.seqs.count( b->seq );
    b->start = a.seqs.start ? min( a.seqs.start[b->seq], 0x7fffffffu ) : 0u;
    return true;
  }
}

// keys that token t of a block's sequence attends
__device__ __forceinline__ uint32_t visible( const Call& a, const Block& b, uint32_t t ) { return min( b.start + t + 1, a.max_keys ); }

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
// =================================================================================================
template<typename T, int NB, bool DECODE>
__global__ __launch_bounds__( 256 ) void attn_pages_f32_kernel( const T* __restrict__ q, T* __restrict__ out, Call a )
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
  if constexpr ( !DECODE ) {
    // rows with a NaN, once more key by key
    float probe = l;
#pragma unroll
    for ( int n = 0; n < NB; n++ ) {
      probe += 0.0f * ( ( acc[n][0] + acc[n][1] ) + ( acc[n][2] + acc[n][3] ) );
    }
    const bool bad = mine && probe != probe;
    uint64_t todo = __builtin_amdgcn_ballot_w64( bad );
    todo = ( todo | todo >> 16 | todo >> 32 | todo >> 48 ) & 0xffff; // columns
    if ( todo != 0 ) {
      const uint32_t keep = ok && !( todo >> c & 1 );
      for ( uint32_t cc = 0; cc < 16; cc++ ) {
        if ( !( todo >> cc & 1 ) ) {
          continue;
        }
        const uint32_t cl = b.col0 + 16 * wave + cc, t = cl / a.gqa, hd = b.h * a.gqa + cl % a.gqa;
        const uint64_t at = (uint64_t)( b.row0 + t ) * n_heads + hd;
        float wm, wl, wacc[4];
        walk_row<T>( q + at * a.size, a.pages, b.seq, kv_off, v_off, a.size, k_begin, min( visible( a, b, t ), k_end ), a.scale_log2e, &wm, &wl, wacc );
        for ( int u = 0; u < 4; u++ ) {
          const uint32_t d = 64 * u + lane;
          if ( d < a.size ) {
            if ( a.splits == 1 ) {
              out[at * a.size + d] = from_f32<T>( wacc[u] / wl );
            } else {
              a.part_out[( at * a.splits + b.split ) * a.size + d] = wacc[u];
            }
          }
        }
        if ( a.splits > 1 && lane == 0 ) {
          a.part_ml[( at * a.splits + b.split ) * 2] = wm;
          a.part_ml[( at * a.splits + b.split ) * 2 + 1] = wl;
        }
      }
      if ( !keep ) {
        return;
      }
    }
  }
  if ( !mine ) {
    return;
  }
  if ( a.splits > 1 ) {
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
    return;
  }
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

// =================================================================================================
// splits of a row added up: wave <-> (query row, head)
// =================================================================================================
template<typename T, bool DECODE>
__global__ __launch_bounds__( 256 ) void pages_merge_kernel( T* __restrict__ out, Call a, uint32_t rows )
{
  const uint32_t lane = threadIdx.x & 63, n_heads = a.n_kv_heads * a.gqa;
  const uint64_t place = (uint64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane( threadIdx.x >> 6 );
  const uint32_t row = (uint32_t)( place / n_heads );
  if ( row >= rows ) {
    return;
  }
  uint32_t keys;
  if constexpr ( DECODE ) {
    keys = min( a.lengths[row], a.max_keys );
  } else {
    const uint32_t seq = packed_sequence( a.seqs, row );
    if ( seq >= a.seqs.batch || a.seqs.count( seq ) <= row - a.seqs.begin( seq ) ) {
      return;
    }
    const uint32_t start = a.seqs.start ? min( a.seqs.start[seq], 0x7fffffffu ) : 0u;
    keys = min( start + ( row - a.seqs.begin( seq ) ) + 1, a.max_keys );
  }
  const uint32_t n = ( keys + a.chunk - 1 ) / a.chunk; // at most a.splits, as max_keys is at most splits * chunk
  if ( n == 0 ) {
    return;
  }
  const float* ml = a.part_ml + place * a.splits * 2;
  const float* part = a.part_out + place * a.splits * a.size;
  float mm = -INFINITY;
  for ( uint32_t s = lane; s < n; s += 64 ) {
    mm = fmaxf( mm, ml[2 * s] );
  }
  mm = wave_max( mm );
  const float mm_safe = mm == -INFINITY ? 0.0f : mm;
  float l = 0.0f, acc[4] = { 0, 0, 0, 0 };
  for ( uint32_t s0 = 0; s0 < n; s0 += 64 ) {
    float w = 0.0f, ls = 0.0f;
    if ( s0 + lane < n ) {
      w = fast_exp2( ml[2 * ( s0 + lane )] - mm_safe );
      ls = ml[2 * ( s0 + lane ) + 1];
    }
    l += wave_sum( w * ls );
    const uint32_t k = min( 64u, n - s0 );
    for ( uint32_t s = 0; s < k; s++ ) {
      const float ws = __shfl( w, (int)s, WAVE );
#pragma unroll
      for ( int u = 0; u < 4; u++ ) {
        const uint32_t d = 64 * u + lane;
        if ( d < a.size ) {
          acc[u] = __builtin_fmaf( part[(uint64_t)( s0 + s ) * a.size + d], ws, acc[u] );
        }
      }
    }
  }
#pragma unroll
  for ( int u = 0; u < 4; u++ ) {
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
  uint64_t bytes;
};

// Keys of a split: whole numbers of 64.  As many splits as bring the launch to four work-groups a CU, of at least 256 keys.
Plan plan_call( bool decode, uint64_t batch, uint64_t rows, uint32_t max_keys, const gh_shape* s )
{
  Plan p {};
  const uint32_t cols = decode ? 16 : 64;
  p.n_blocks = decode ? ( s->gqa_size + cols - 1 ) / cols : 0;
  const uint64_t blocks = decode ? batch * p.n_blocks : std::min<uint64_t>( ( rows * s->gqa_size + cols - 1 ) / cols + batch, rows * s->gqa_size );
  p.blocks = (uint32_t)blocks;
  const uint64_t groups = blocks * s->n_kv_heads;
  uint64_t splits = std::max<uint64_t>( 1, std::min<uint64_t>( 4ull * (uint64_t)cu_count() / groups, ( max_keys + 255 ) / 256 ) );
  p.chunk = (uint32_t)( ( ( max_keys + splits - 1 ) / splits + 63 ) / 64 * 64 );
  p.splits = ( max_keys + p.chunk - 1 ) / p.chunk;
  p.bytes = p.splits == 1 ? 0 : rows * s->n_heads * p.splits * ( s->head_size + 2 ) * sizeof( float );
  return p;
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

template<typename T, bool DECODE>
int launch( const Plan& p, const Call& a, const void* q, void* out, uint64_t rows, hipStream_t st )
{
  launch_f32<T, DECODE>( p, a, q, out, st );
  GH_LAUNCH_CHECK();
  if ( p.splits > 1 ) {
    pages_merge_kernel<T, DECODE><<<(unsigned)( ( rows * a.n_kv_heads * a.gqa + 3 ) / 4 ), 256, 0, st>>>( static_cast<T*>( out ), a, (uint32_t)rows );
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
  const Plan p = plan_call( DECODE, batch, rows, max_keys, s );
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
  return !shape_ok( shape ) || batch == 0 || max_length == 0 ? 0 : plan_call( true, batch, batch, max_length, shape ).bytes;
}

int gh_attn_decode_paged( const void* q, const gh_pages* pages, const uint32_t* lengths_dev, void* xb, uint64_t batch, uint32_t max_length, const gh_shape* shape,
                          gh_dtype dt, void* workspace, uint64_t workspace_bytes, gh_stream stream )
{
  return attn_pages<true>( "gh_attn_decode_paged", q, pages, lengths_dev, nullptr, nullptr, xb, batch, batch, max_length, shape, dt, workspace, workspace_bytes, stream );
}

uint64_t gh_attn_packed_workspace( uint64_t batch, uint64_t n_tokens, uint32_t max_keys, const gh_shape* shape, gh_dtype dt )
{
  return !shape_ok( shape ) || batch == 0 || n_tokens == 0 || max_keys == 0 ? 0 : plan_call( false, batch, n_tokens, max_keys, shape ).bytes;
}

int gh_attn_packed( const void* q, const gh_pages* pages, const uint32_t* first_dev, const uint32_t* start_pos_dev, void* xb, uint64_t batch, uint64_t n_tokens,
                    uint32_t max_keys, const gh_shape* shape, gh_dtype dt, void* workspace, uint64_t workspace_bytes, gh_stream stream )
{
  return attn_pages<false>( "gh_attn_packed", q, pages, nullptr, first_dev, start_pos_dev, xb, batch, n_tokens, max_keys, shape, dt, workspace, workspace_bytes, stream );
}

} // extern "C"
