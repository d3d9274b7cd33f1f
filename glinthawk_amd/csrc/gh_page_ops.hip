// What a cache in pages needs besides its attention: the rows of packed tokens, and pages copied within their pool.
#include "gh_pages.h"

#include <algorithm>
#include <new>
#include <vector>

namespace gh {
namespace {

// thread <-> packed token, which finds its sequence by bisection: the last one that begins at or before it.  Bound by latency (a launch of 5 us).
__global__ __launch_bounds__( 256 ) void page_rows_kernel( Pages p, Packed s, void** __restrict__ rows_out, uint32_t* __restrict__ pos_out )
{
  const uint32_t t = blockIdx.x * 256 + threadIdx.x;
  if ( t >= s.tokens ) {
    return;
  }
  const uint32_t low = last_at_most( s.batch, t, [&]( uint32_t i ) { return s.begin( i ); } );
  const bool has = s.begin( low ) <= t && t < s.begin( low + 1 );
  const uint64_t pos = ( has && s.start ? (uint64_t)s.start[low] : 0 ) + ( has ? t - s.begin( low ) : 0 );
  void* row = nullptr;
  if ( has && pos < p.reach() ) {
    const uint32_t page = p.table[(uint64_t)low * p.table_stride + ( (uint32_t)pos >> p.shift )];
    if ( page <= p.last ) {
      row = const_cast<char*>( p.pool ) + page * p.stride + (uint64_t)( (uint32_t)pos & ( ( 1u << p.shift ) - 1 ) ) * p.row_bytes;
    }
  }
  if ( rows_out ) {
    rows_out[t] = row;
  }
  if ( pos_out ) {
    pos_out[t] = row ? (uint32_t)pos : 0u;
  }
}

// grid: (pieces of a page, pairs, layers); P: 16 bytes, or 2 where addresses or sizes are not multiples of 16 (1 where they are odd)
// Bound by the bytes: 1999 pages of 64 KB in 4 layers 187 us, 5.6 TB/s in and out; by its launch where there are few: 5 such pages in 10 layers 3 us.
template<typename P>
__global__ __launch_bounds__( 256 ) void copy_pages_kernel( char* pool, uint64_t stride, uint64_t bytes, uint32_t n_pages, uint64_t layer_stride,
                                                          const uint32_t* __restrict__ pairs, uint32_t n_pairs )
{
  for ( uint32_t j = blockIdx.y; j < n_pairs; j += gridDim.y ) {
    const uint32_t from = pairs[2 * (uint64_t)j], to = pairs[2 * (uint64_t)j + 1];
    if ( from >= n_pages || to >= n_pages ) {
      continue;
    }
    const P* src = reinterpret_cast<const P*>( pool + blockIdx.z * layer_stride + from * stride );
    P* dst = reinterpret_cast<P*>( pool + blockIdx.z * layer_stride + to * stride );
    const uint64_t n = bytes / sizeof( P );
    for ( uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256 ) {
      dst[i] = src[i];
    }
  }
}

int check_copy( const char* op, const void* pool, uint64_t stride, uint64_t bytes, uint32_t n_pages, uint64_t layers, uint64_t layer_stride, const uint32_t* pairs,
                uint64_t n_pairs )
{
  GH_REQUIRE( pool && pairs, "%s: NULL pointer", op );
  GH_REQUIRE( n_pages > 0 && bytes > 0 && stride >= bytes && stride < 1ull << 40, "%s: bad pages", op );
  GH_REQUIRE( layers <= 65535 && ( layers == 1 || layer_stride < 1ull << 47 ), "%s: too many layers, or too far apart", op );
  GH_REQUIRE( n_pairs <= 0x7fffffffull, "%s: too many pairs", op );
  GH_REQUIRE( reinterpret_cast<uintptr_t>( pairs ) % 4 == 0, "%s: pairs are not aligned to their numbers", op );
  // a layer that begins inside another's pages: what one copies the other could write
  const uint64_t span = ( n_pages - 1 ) * stride + bytes;
  GH_REQUIRE( layers == 1 || layer_stride >= span || ( layer_stride >= bytes && stride >= layers * layer_stride - ( layer_stride - bytes ) ),
              "%s: layers of %llu bytes lie %llu apart", op, (unsigned long long)span, (unsigned long long)layer_stride );
  return GH_OK;
}

int copy_pairs( void* pool, uint64_t stride, uint64_t bytes, uint32_t n_pages, uint64_t layers, uint64_t layer_stride, const uint32_t* pairs_dev, uint64_t n_pairs,
                hipStream_t st )
{
  const uint64_t places = reinterpret_cast<uintptr_t>( pool ) | stride | bytes | ( layers > 1 ? layer_stride : 0 );
  auto launch = [&]( auto piece ) {
    using P = decltype( piece );
    const uint64_t pieces = ( bytes / sizeof( P ) + 255 ) / 256;
    const dim3 grid( (unsigned)std::min<uint64_t>( pieces, 64 ), (unsigned)std::min<uint64_t>( n_pairs, 65535 ), (unsigned)layers );
    copy_pages_kernel<P><<<grid, 256, 0, st>>>( static_cast<char*>( pool ), stride, bytes, n_pages, layer_stride, pairs_dev, (uint32_t)n_pairs );
  };
  if ( places % 16 == 0 ) {
    launch( uint4 {} );
  } else if ( places % 2 == 0 ) {
    launch( uint16_t {} );
  } else {
    launch( uint8_t {} );
  }
  GH_LAUNCH_CHECK();
  return GH_OK;
}

} // namespace
} // namespace gh

using namespace gh;

extern "C" {

int gh_page_rows( const gh_pages* pages, const uint32_t* first_dev, const uint32_t* start_pos_dev, uint64_t batch, uint64_t n_tokens, uint32_t kv_dim,
                  void** token_rows_out, uint32_t* pos_out, gh_dtype dt, gh_stream stream )
{
  Pages p;
  if ( n_tokens != 0 ) { // what can be said without a device is said first
    if ( int rc = check_pages( "gh_page_rows", pages, kv_dim, dt, &p ) ) {
      return rc;
    }
    GH_REQUIRE( first_dev, "gh_page_rows: NULL table" );
    GH_REQUIRE( batch > 0 && batch <= 0x7ffffffeull && n_tokens <= 0x7fffffffull, "gh_page_rows: bad shape" );
  }
  if ( int rc = ensure_init() ) {
    return rc;
  }
  if ( n_tokens == 0 ) {
    return GH_OK;
  }
  const Packed s { first_dev, start_pos_dev, (uint32_t)batch, (uint32_t)n_tokens };
  page_rows_kernel<<<(unsigned)( ( n_tokens + 255 ) / 256 ), 256, 0, as_stream( stream )>>>( p, s, token_rows_out, pos_out );
  GH_LAUNCH_CHECK();
  return GH_OK;
}

int gh_copy_pages( void* pool, uint64_t page_stride, uint64_t page_bytes, uint32_t n_pages, uint64_t layers, uint64_t layer_stride, const uint32_t* pairs_dev,
                   uint64_t n_pairs, gh_stream stream )
{
  if ( n_pairs != 0 && layers != 0 ) {
    if ( int rc = check_copy( "gh_copy_pages", pool, page_stride, page_bytes, n_pages, layers, layer_stride, pairs_dev, n_pairs ) ) {
      return rc;
    }
  }
  if ( int rc = ensure_init() ) {
    return rc;
  }
  if ( n_pairs == 0 || layers == 0 ) {
    return GH_OK;
  }
  return copy_pairs( pool, page_stride, page_bytes, n_pages, layers, layer_stride, pairs_dev, n_pairs, as_stream( stream ) );
}

int gh_copy_pages_host( void* pool, uint64_t page_stride, uint64_t page_bytes, uint32_t n_pages, uint64_t layers, uint64_t layer_stride, const uint32_t* pairs_host,
                        uint64_t n_pairs, gh_stream stream )
{
  if ( n_pairs != 0 && layers != 0 ) {
    if ( int rc = check_copy( "gh_copy_pages_host", pool, page_stride, page_bytes, n_pages, layers, layer_stride, pairs_host, n_pairs ) ) {
      return rc;
    }
    std::vector<uint32_t> written;
    try {
      written.resize( n_pairs );
    } catch ( const std::bad_alloc& ) {
      return fail( GH_ERR_OOM, "gh_copy_pages_host: no memory to check %llu pairs", (unsigned long long)n_pairs );
    }
    for ( uint64_t j = 0; j < n_pairs; j++ ) {
      GH_REQUIRE( pairs_host[2 * j] < n_pages && pairs_host[2 * j + 1] < n_pages, "gh_copy_pages_host: pair %llu, %u to %u, of %u pages", (unsigned long long)j,
                  pairs_host[2 * j], pairs_host[2 * j + 1], n_pages );
      written[j] = pairs_host[2 * j + 1];
    }
    std::sort( written.begin(), written.end() );
    for ( uint64_t j = 1; j < n_pairs; j++ ) {
      GH_REQUIRE( written[j] != written[j - 1], "gh_copy_pages_host: page %u is written twice", written[j] );
    }
    for ( uint64_t j = 0; j < n_pairs; j++ ) {
      GH_REQUIRE( !std::binary_search( written.begin(), written.end(), pairs_host[2 * j] ), "gh_copy_pages_host: page %u is read and written", pairs_host[2 * j] );
    }
  }
  if ( int rc = ensure_init() ) {
    return rc;
  }
  if ( n_pairs == 0 || layers == 0 ) {
    return GH_OK;
  }
  constexpr uint64_t PART = STAGE_SLOT_BYTES / 8; // pairs of a staging slot; the pages of different pairs are apart, so parts may follow each other in any order
  hipStream_t st = as_stream( stream );
  if ( st != nullptr ) { // a graph would copy the pairs from the staging slot again when that holds something else
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    GH_HIP( hipStreamIsCapturing( st, &capture ) );
    GH_REQUIRE( capture == hipStreamCaptureStatusNone, "gh_copy_pages_host: the stream is being captured into a graph, which takes pairs in device memory" );
  }
  for ( uint64_t j = 0; j < n_pairs; j += PART ) {
    const uint64_t n = std::min( PART, n_pairs - j );
    StageScope scope( st );
    void* dev = nullptr;
    if ( int rc = stage_table( pairs_host + 2 * j, n * 8, st, &dev ) ) {
      return rc;
    }
    if ( int rc = copy_pairs( pool, page_stride, page_bytes, n_pages, layers, layer_stride, static_cast<const uint32_t*>( dev ), n, st ) ) {
      return rc;
    }
    if ( int rc = scope.finish() ) {
      return rc;
    }
  }
  return GH_OK;
}

} // extern "C"
