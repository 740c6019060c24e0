// What a failed runtime call leaves behind (linked with fake_runtime.cc). Prints the
// number of checks that failed.
#include <stdio.h>
#include <string.h>

#include "common.cuh"

extern "C" int fake_last;

static int launches_well() {
    OFB_CHECK_LAUNCH("a launch");
    return OFB_OK;
}

int main() {
    int bad = 0;
    fake_last = cudaErrorInvalidValue;  // a call was refused, and its caller reports it
    bad += ofb::cuda_status(cudaErrorInvalidValue, "refused call") != OFB_ECUDA;
    bad += strstr(ofb_last_error(), "refused call") == nullptr;
    bad += launches_well() != OFB_OK;  // the next call does not
    fake_last = cudaErrorMemoryAllocation;
    bad += ofb::cuda_status(cudaErrorMemoryAllocation, "allocation") != OFB_ENOMEM;
    bad += launches_well() != OFB_OK;
    fake_last = cudaErrorInvalidConfiguration;  // a launch that failed itself is reported, once
    bad += launches_well() != OFB_ECUDA;
    bad += launches_well() != OFB_OK;
    printf("%d\n", bad);
    return 0;
}
