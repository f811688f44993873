#include "attention.cuh"
