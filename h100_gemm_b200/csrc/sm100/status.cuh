// Codes the kernels write to the device's status word.
#pragma once

namespace b200 {

// Device status codes written to the status word when a bounded wait gives up.
enum DeviceStatus : unsigned int {
  kStatusOk = 0,
  kStatusProducerTimeout = 1,   // producer waited for empty[s]
  kStatusMmaFullTimeout = 2,    // MMA issuer waited for full[s]
  kStatusMmaTmemTimeout = 3,    // MMA issuer waited for tmem_empty[a]
  kStatusEpilogueTimeout = 4,   // epilogue waited for tmem_full[a]
  kStatusStreamKTimeout = 5,    // stream-K finisher waited for another worker's partial tile
  kStatusSelfTestTimeout = 9,   // the bounded-wait self-test (an mbarrier nothing arrives on)
};

}  // namespace b200
