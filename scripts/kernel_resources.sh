#!/bin/bash
# Registers / scratch / LDS of every kernel in the library (compile-only, runs without a GPU).
cd "$(dirname "$0")/.."
for unit in sp_knn sp_dense; do
  /opt/rocm/bin/hipcc --offload-arch=gfx950 -O3 -std=c++17 -munsafe-fp-atomics -Xclang -target-feature -Xclang -packed-fp32-ops -fPIC -Wno-unused-function -I include \
    -Rpass-analysis=kernel-resource-usage -c similaripy_amd/csrc/$unit.hip -o /tmp/${unit}_res.o 2>&1 |
    grep -E "Function Name|VGPRs:|ScratchSize|Occupancy|SGPRs:" | sed 's/.*remark: [^ ]* *//' | paste - - - - - | grep -v "SGPRs: 0 "
done
