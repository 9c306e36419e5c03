// What the operators outside context.cc use of a context and its stores.
#ifndef MMR_CSRC_CONTEXT_ACCESS_H_
#define MMR_CSRC_CONTEXT_ACCESS_H_

#include <hip/hip_runtime_api.h>

#include <initializer_list>
#include <memory>
#include <mutex>

#include "common.h"

namespace mmr {

// An operator's handle, owned by the context; destroyed with it at the latest.
struct Attachment {
  virtual ~Attachment() = default;
  mmr_context* owner = nullptr;
};

// The context's lock, for the length of an entry point; notes that the call may queue work on the stream.
class ContextLock {
 public:
  explicit ContextLock(mmr_context* ctx);

 private:
  std::unique_lock<std::mutex> lock_;
};

int context_use_device(mmr_context* ctx);  // the context's GPU becomes current
hipStream_t context_stream(mmr_context* ctx);
int context_refuse_capture(mmr_context* ctx, const char* what);
int context_wait(mmr_context* ctx);  // host waits for the stream
void context_count(mmr_context* ctx, int64_t launches);
// rolling hash of the operation stream (MMR_CHECK_INVARIANTS)
void context_hash(mmr_context* ctx, uint64_t kind, std::initializer_list<uint64_t> values);
// Device memory for tables, from and to the context's block pool; its next user is ordered behind the stream.
int context_take_block(mmr_context* ctx, size_t bytes, char** out, size_t* capacity);
void context_give_block(mmr_context* ctx, char* block, size_t capacity);
// Stream-ordered; `host` may be reused when the call returns.  Not while the stream is capturing.
int context_upload(mmr_context* ctx, void* device, const void* host, size_t bytes);

void context_attach(mmr_context* ctx, std::unique_ptr<Attachment> a);
void context_detach(mmr_context* ctx, Attachment* a);  // destroys it

// Counts what may change where the buffers of watched stores are: frees, offloads, reloads.
uint64_t context_store_epoch(mmr_context* ctx);
void context_watch(mmr_store* store);
mmr_store* context_find_store(mmr_context* ctx, int64_t id);  // null if it was freed
// The store is this context's and on the device.
int context_check_store(mmr_context* ctx, const mmr_store* store, const char* what);
const Side& store_side(const mmr_store* store);
const std::string& store_key(const mmr_store* store);
int64_t store_ordinal(const mmr_store* store);
char* store_tile(const mmr_store* store, int64_t k);
bool store_tiles_overlap(const mmr_store* store);  // adopted buffers that lie over one another, as replicas in one do

}  // namespace mmr

#endif  // MMR_CSRC_CONTEXT_ACCESS_H_
