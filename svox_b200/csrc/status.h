// The anomaly words of the translation units that have one of their own (a __device__ variable
// belongs to one): svoxb_device_status returns the largest of all.
#pragma once

namespace svoxb {
int status_of_recurrence(int clear, int* word);
int status_of_rays(int clear, int* word);
int status_of_records(int clear, int* word);
}  // namespace svoxb
