// What the kernels over a paged cache share: the address of a token's row, the sequence and tokens of a work-group's block, and the checks of a
// description of pages.
#pragma once

#include "gh_common.h"

namespace gh {

struct Pages
{
  const char* pool;
  uint64_t stride; // bytes from page to page
  uint32_t last;   // number of the last page
  uint32_t shift;  // page_tokens = 1 << shift
  const uint32_t* table;
  uint32_t table_stride;
  uint32_t row_bytes;

  // a page number that the pool does not have reads as its last page
  __host__ __device__ __forceinline__ const char* page( uint32_t seq, uint32_t index ) const
  {
    const uint32_t number = table[(uint64_t)seq * table_stride + index];
    return pool + ( number < last ? number : last ) * stride;
  }
  __host__ __device__ __forceinline__ const char* row( uint32_t seq, uint32_t key ) const
  {
    return page( seq, key >> shift ) + (uint64_t)( key & ( ( 1u << shift ) - 1 ) ) * row_bytes;
  }
  // keys that the table reaches (below 2^31, see check_pages)
  __host__ __device__ __forceinline__ uint32_t reach() const { return table_stride << shift; }
};

// Checks a caller's description and gives the kernels' form of it.
inline int check_pages( const char* op, const gh_pages* p, uint64_t kv_dim, gh_dtype dt, Pages* out )
{
  GH_REQUIRE( dt == GH_F16 || dt == GH_F32 || dt == GH_BF16, "%s: unsupported dtype %d", op, (int)dt );
  GH_REQUIRE( p != nullptr && p->pool && p->table, "%s: NULL pages", op );
  const uint64_t size = dtype_size( dt );
  GH_REQUIRE( kv_dim > 0 && kv_dim <= 1u << 24, "%s: bad kv_dim", op );
  GH_REQUIRE( p->n_pages > 0 && p->table_stride > 0, "%s: no pages", op );
  GH_REQUIRE( p->page_tokens > 0 && ( p->page_tokens & ( p->page_tokens - 1 ) ) == 0, "%s: a page of %u tokens is no power of two", op, p->page_tokens );
  const uint64_t page_bytes = 2 * kv_dim * size * p->page_tokens;
  GH_REQUIRE( page_bytes < 1ull << 31, "%s: a page of %llu bytes (2 GiB and more)", op, (unsigned long long)page_bytes );
  GH_REQUIRE( p->page_stride >= page_bytes && p->page_stride % size == 0 && p->page_stride < 1ull << 40, "%s: pages of %llu bytes lie %llu apart", op,
              (unsigned long long)page_bytes, (unsigned long long)p->page_stride );
  GH_REQUIRE( reinterpret_cast<uintptr_t>( p->pool ) % size == 0 && reinterpret_cast<uintptr_t>( p->table ) % 4 == 0, "%s: pool or table is not aligned to its elements", op );
  GH_REQUIRE( (uint64_t)p->table_stride * p->page_tokens < 1ull << 31, "%s: a table that reaches 2^31 tokens", op );
  *out = { static_cast<const char*>( p->pool ), p->page_stride, p->n_pages - 1, (uint32_t)__builtin_ctz( p->page_tokens ), p->table, p->table_stride,
           (uint32_t)( 2 * kv_dim * size ) };
  return GH_OK;
}

// ---- packed sequences ---------------------------------------------------------------------------
struct Packed
{
  const uint32_t* first; // batch + 1
  const uint32_t* start; // batch, or NULL: all 0
  uint32_t batch;
  uint32_t tokens; // rows there are, whatever `first` says

  __device__ __forceinline__ uint32_t begin( uint32_t i ) const { return min( first[i], tokens ); }
  __device__ __forceinline__ uint32_t count( uint32_t i ) const
  {
    const uint32_t b = begin( i ), e = begin( i + 1 );
    return e > b ? e - b : 0;
  }
  // position of its first token, so that sums of it and a number of tokens (at most 2^24) stay below 2^32; a table reaches no position beyond
  __device__ __forceinline__ uint32_t begin_pos( uint32_t i ) const { return start ? min( start[i], 0x7fffffffu ) : 0u; }
};

// sum or maximum over the wave, in every lane: rows of 16 lanes by DPP, the four rows by lane reads
template<typename F>
__device__ __forceinline__ uint32_t wave_all( uint32_t v, F f )
{
  v = f( v, (uint32_t)__builtin_amdgcn_update_dpp( 0, (int)v, 0xB1, 0xF, 0xF, true ) );
  v = f( v, (uint32_t)__builtin_amdgcn_update_dpp( 0, (int)v, 0x4E, 0xF, 0xF, true ) );
  v = f( v, (uint32_t)__builtin_amdgcn_update_dpp( 0, (int)v, 0x141, 0xF, 0xF, true ) );
  v = f( v, (uint32_t)__builtin_amdgcn_update_dpp( 0, (int)v, 0x140, 0xF, 0xF, true ) );
  return f( f( (uint32_t)__builtin_amdgcn_readlane( (int)v, 0 ), (uint32_t)__builtin_amdgcn_readlane( (int)v, 16 ) ),
            f( (uint32_t)__builtin_amdgcn_readlane( (int)v, 32 ), (uint32_t)__builtin_amdgcn_readlane( (int)v, 48 ) ) );
}
__device__ __forceinline__ uint32_t wave_sum_u32( uint32_t v )
{
  return wave_all( v, []( uint32_t a, uint32_t b ) { return a + b; } );
}
__device__ __forceinline__ uint32_t wave_max_u32( uint32_t v )
{
  return wave_all( v, []( uint32_t a, uint32_t b ) { return a > b ? a : b; } );
}

// The last sequence i with key( i ) <= value, for keys that do not fall; 0 if there is none.
template<typename Key>
__device__ __forceinline__ uint32_t last_at_most( uint32_t batch, uint32_t value, Key key )
{
  uint32_t low = 0, high = batch;
  while ( high - low > 1 ) {
    const uint32_t middle = ( low + high ) / 2;
    if ( key( middle ) <= value ) {
      low = middle;
    } else {
      high = middle;
    }
  }
  return low;
}

// A sequence as packed_block found it
struct PackedBlock
{
  uint32_t seq, block;
  uint32_t row0, tokens, start; // of the sequence
};

// Block number -> (sequence, block of the sequence), by a whole wave.  A sequence of n tokens with `gqa` columns each has ceil(n gqa / columns) blocks.  Blocks are
// numbered by falling level, which is the block's place in its sequence plus the blocks that the sequence's start position would be, so that the ones with the most
// keys come first and a launch does not end on a long one.  The level of a number is found by bisection over how many blocks lie at a level and above, a sum over the
// sequences.  False: no such block.
// Every block reads all sequences for that, so where there are many numbers go by the sequences' places: sequence i has those from floor(first[i] gqa / columns) + i on,
// at least as many as it has blocks, and its last block comes first.  In order and by place, us: f16, 64 heads on 8 of 128, 1 to 300 tokens each: 65 sequences 175 and
// 148, 200 564 and 385, 500 1858 and 927; 200 of one token behind 1000 keys 143 and 123, 2000 2590 and 1017; 64 and fewer are kept in registers.
// fp32, 12 heads of 64, where a block takes longer and fewer run at a time: one token behind 0 to 2000 keys, 100 sequences 148 and 170, 200 281 and 295, 500 908 and 665;
// 1 to 300 tokens, 200 sequences 281 and 207.
__host__ __device__ constexpr uint32_t most_ordered( uint32_t columns ) { return columns == 128 ? 64 : 256; } // 128: of the 16-bit kernel
// numbers of blocks there may be: a block has a column, and all but the last of a sequence are full
__host__ __device__ constexpr uint64_t most_blocks( uint64_t all_columns, uint64_t batch, uint32_t columns )
{
  return ( all_columns + columns - 1 ) / columns + batch < all_columns ? ( all_columns + columns - 1 ) / columns + batch : all_columns;
}
__device__ __forceinline__ bool packed_block( const Packed& s, uint32_t gqa, uint32_t columns, uint32_t number, PackedBlock* found )
{
  const uint32_t lane = threadIdx.x & 63;
  auto blocks_of = [&]( uint32_t tokens ) { return (uint32_t)( ( (uint64_t)tokens * gqa + columns - 1 ) / columns ); };
  if ( s.batch > most_ordered( columns ) ) {
    // where there are fewer columns than such numbers, a number is a column's, and the block's that it begins
    const bool by_column = most_blocks( (uint64_t)s.tokens * gqa, s.batch, columns ) == (uint64_t)s.tokens * gqa;
    auto slot = [&]( uint32_t i ) { return by_column ? s.begin( i ) * gqa : (uint32_t)( (uint64_t)s.begin( i ) * gqa / columns ) + i; };
    const uint32_t i = last_at_most( s.batch, number, slot ), n = blocks_of( s.count( i ) ), place = number - slot( i );
    *found = { i, by_column ? place / columns : n - 1 - place, s.begin( i ), s.count( i ), s.begin_pos( i ) };
    return slot( i ) <= number && ( by_column ? place < s.count( i ) * gqa && place % columns == 0 : place < n );
  }
  auto blocks = [&]( uint32_t i ) { return i < s.batch ? blocks_of( s.count( i ) ) : 0u; };
  auto level_of = [&]( uint32_t start ) { return (uint32_t)min( (uint64_t)start * gqa / columns, (uint64_t)0x3fffffff ); }; // of a sequence's first block
  auto level0 = [&]( uint32_t i ) { return i < s.batch ? level_of( s.begin_pos( i ) ) : 0u; };
  // what there is to know of the first 64 sequences is read once, and kept
  const uint32_t at = min( lane, s.batch - 1 ), my_row0 = s.begin( at ), my_tokens = s.count( at ), my_start = s.begin_pos( at );
  if ( s.batch == 1 ) {
    const uint32_t n = blocks_of( my_tokens );
    *found = { 0, n - 1 - number, my_row0, my_tokens, my_start };
    return number < n;
  }
  const uint32_t mine = lane < s.batch ? blocks_of( my_tokens ) : 0, mine0 = level_of( my_start );
  uint32_t most = mine == 0 ? 0 : mine0 + mine;
  for ( uint32_t i = 64 + lane; i < s.batch; i += 64 ) {
    const uint32_t n = blocks( i );
    most = max( most, n == 0 ? 0 : level0( i ) + n );
  }
  most = wave_max_u32( most );
  auto above = [&]( uint32_t level ) { // blocks at `level` and beyond
    uint32_t n = min( mine, mine0 + mine > level ? mine0 + mine - level : 0u );
    for ( uint32_t i = 64 + lane; i < s.batch; i += 64 ) {
      const uint32_t b = blocks( i ), end = level0( i ) + b;
      n += min( b, end > level ? end - level : 0u );
    }
    return wave_sum_u32( n );
  };
  if ( above( 0 ) <= number ) {
    return false;
  }
  uint32_t low = 0, high = most; // above( low ) > number >= above( high )
  while ( high - low > 1 ) {
    const uint32_t middle = ( low + high ) / 2;
    if ( above( middle ) > number ) {
      low = middle;
    } else {
      high = middle;
    }
  }
  uint32_t rank = number - above( low + 1 ); // among the sequences that have a block at this level
  for ( uint32_t i0 = 0; i0 < s.batch; i0 += 64 ) {
    const uint32_t first = i0 == 0 ? mine0 : level0( i0 + lane ), n_blocks = i0 == 0 ? mine : blocks( i0 + lane );
    const uint64_t have = __builtin_amdgcn_ballot_w64( first <= low && low < first + n_blocks );
    const uint32_t n = __popcll( have );
    if ( rank < n ) {
      // the lane whose set bit has `rank` set bits below it
      const uint64_t hit = __builtin_amdgcn_ballot_w64( ( have >> lane & 1 ) && (uint32_t)__popcll( have & ( ( 1ull << lane ) - 1 ) ) == rank );
      const uint32_t which = (uint32_t)__builtin_ctzll( hit );
      found->seq = i0 + which;
      found->block = low - (uint32_t)__builtin_amdgcn_readlane( (int)first, (int)which );
      if ( i0 == 0 ) {
        found->row0 = (uint32_t)__builtin_amdgcn_readlane( (int)my_row0, (int)which );
        found->tokens = (uint32_t)__builtin_amdgcn_readlane( (int)my_tokens, (int)which );
        found->start = (uint32_t)__builtin_amdgcn_readlane( (int)my_start, (int)which );
      } else {
        found->row0 = s.begin( found->seq );
        found->tokens = s.count( found->seq );
        found->start = s.begin_pos( found->seq );
      }
      return true;
    }
    rank -= n;
  }
  return false;
}

// The sequence a packed row belongs to, by a whole wave; batch: none.
__device__ __forceinline__ uint32_t packed_sequence( const Packed& s, uint32_t row )
{
  uint32_t i;
  if ( s.batch <= 64 ) { // as many sequences as end at or before it lie in front
    const uint32_t lane = threadIdx.x & 63;
    i = __popcll( __builtin_amdgcn_ballot_w64( lane < s.batch && s.begin( lane + 1 ) <= row ) );
  } else {
    i = last_at_most( s.batch, row, [&]( uint32_t k ) { return s.begin( k ); } );
  }
  return i < s.batch && s.begin( i ) <= row && row < s.begin( i + 1 ) ? i : s.batch;
}

} // namespace gh
