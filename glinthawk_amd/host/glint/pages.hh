// Bookkeeping of a cache in pages (gh_pages of include/glint_hip.h): which pages of a pool the contexts have, in order, and how many contexts a page has.  A fork
// shares its parent's pages; the first to write into a shared last page gets a copy of it.  Integers only: the copies that a call asks for come back as pairs
// (source, destination), for gh_copy_pages to carry out before anything is written to or read from the pages that moved.
//   - the free page with the lowest number is taken first
//   - a call that cannot be served, for want of pages or of memory, changes nothing
//   - the pairs of one call never name a page twice among the destinations, nor one as source and destination.  That holds for pairs of several calls
//     only while nothing is released or compacted between them, so they are carried out first
// No counterpart in the reference, whose contexts are one run of rows each.
#pragma once

#include <algorithm>
#include <cstdint>
#include <mutex>
#include <optional>
#include <unordered_map>
#include <utility>
#include <vector>

namespace glint {

class PageBook
{
public:
  using Pair = std::pair<uint32_t, uint32_t>; // source, destination
  struct Context
  {
    std::vector<uint32_t> pages {};
    uint64_t length { 0 }; // tokens
  };

  PageBook( const uint32_t n_pages, const uint32_t page_tokens )
    : page_tokens_( page_tokens )
    , users_( n_pages, 0 )
    , n_free_( n_pages )
  {
  }

  // Room for `tokens` more tokens of a context, which begins here if it is not known; the copies to make, or nothing if the pages do not suffice.
  std::optional<std::vector<Pair>> extend( const uint64_t id, const uint64_t tokens )
  {
    std::lock_guard lock { mutex_ };
    auto known = contexts_.find( id );
    const uint64_t length = known == contexts_.end() ? 0 : known->second.length;
    const uint64_t have = known == contexts_.end() ? 0 : known->second.pages.size();
    if ( tokens > MOST_TOKENS || length + tokens > MOST_TOKENS ) {
      return std::nullopt;
    }
    const bool copy = tokens > 0 && length % page_tokens_ != 0 && users_[known->second.pages.back()] > 1;
    const uint64_t want = ( length + tokens + page_tokens_ - 1 ) / page_tokens_ - have;
    if ( want + ( copy ? 1 : 0 ) > n_free_ ) {
      return std::nullopt;
    }
    std::vector<Pair> pairs;
    pairs.reserve( 1 ); // what could fail comes before the first change
    if ( known == contexts_.end() ) {
      Context fresh;
      fresh.pages.reserve( want );
      known = contexts_.emplace( id, std::move( fresh ) ).first;
    } else {
      known->second.pages.reserve( have + want );
    }
    auto& context = known->second;
    if ( copy ) {
      const uint32_t old = context.pages.back();
      context.pages.back() = take();
      users_[old]--;
      pairs.emplace_back( old, context.pages.back() );
    }
    for ( uint64_t i = 0; i < want; i++ ) {
      context.pages.push_back( take() );
    }
    context.length = length + tokens;
    return pairs;
  }

  // `child` begins with all that `parent` has; false: no such parent, or the child is known already
  bool fork( const uint64_t parent, const uint64_t child )
  {
    std::lock_guard lock { mutex_ };
    const auto from = contexts_.find( parent );
    if ( from == contexts_.end() || contexts_.count( child ) != 0 ) {
      return false;
    }
    const auto& begun = contexts_.emplace( child, Context { from->second } ).first->second; // (what could fail)
    for ( const uint32_t p : begun.pages ) {
      users_[p]++;
    }
    return true;
  }

  bool release( const uint64_t id )
  {
    std::lock_guard lock { mutex_ };
    const auto it = contexts_.find( id );
    if ( it == contexts_.end() ) {
      return false;
    }
    for ( const uint32_t p : it->second.pages ) {
      if ( --users_[p] == 0 ) {
        give( p );
      }
    }
    contexts_.erase( it );
    return true;
  }

  // Pages in use move to the lowest numbers; the copies to make.  Every context's line may have changed.
  std::vector<Pair> compact()
  {
    std::lock_guard lock { mutex_ };
    const uint32_t used = static_cast<uint32_t>( users_.size() - n_free_ );
    std::vector<uint32_t> to( n_free_ ); // of pages from `used` on
    std::vector<Pair> pairs;
    pairs.reserve( static_cast<size_t>( std::count_if( users_.begin() + used, users_.end(), []( const uint32_t n ) { return n != 0; } ) ) );
    for ( uint32_t p = used; p < users_.size(); p++ ) { // (nothing fails from here on)
      if ( users_[p] != 0 ) {
        const uint32_t place = take(); // below `used`: as many places are free there as pages are in use beyond
        users_[place] = users_[p];
        users_[p] = 0;
        give( p );
        pairs.emplace_back( p, place );
        to[p - used] = place;
      }
    }
    for ( auto& [id, context] : contexts_ ) {
      for ( uint32_t& p : context.pages ) {
        p = p < used ? p : to[p - used];
      }
    }
    return pairs;
  }

  std::optional<Context> context( const uint64_t id ) const
  {
    std::lock_guard lock { mutex_ };
    const auto it = contexts_.find( id );
    return it == contexts_.end() ? std::nullopt : std::optional<Context> { it->second };
  }

  [[nodiscard]] uint64_t free() const
  {
    std::lock_guard lock { mutex_ };
    return n_free_;
  }

private:
  static constexpr uint64_t MOST_TOKENS = ( 1ull << 31 ) - 1; // positions are 32 bits wide

  uint32_t take()
  {
    while ( users_[lowest_] != 0 ) {
      lowest_++;
    }
    users_[lowest_] = 1;
    n_free_--;
    return lowest_++;
  }
  void give( const uint32_t p )
  {
    n_free_++;
    lowest_ = std::min( lowest_, p );
  }

  mutable std::mutex mutex_ {};
  const uint64_t page_tokens_;
  std::vector<uint32_t> users_; // contexts a page has; 0: it is free
  uint32_t n_free_;
  uint32_t lowest_ { 0 }; // no page below is free
  std::unordered_map<uint64_t, Context> contexts_ {};
};

} // namespace glint
